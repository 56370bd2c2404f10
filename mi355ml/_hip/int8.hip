// Products of 8-bit matrices, and the quantiser that makes them.
//
//   quantize:  s[i] = f32(max_k |x[i,k]| / 127),  q[i,k] = rne(x[i,k] / s[i])
//   product:   y[i,j] = (sum_k xq[i,k] wq[j,k]) xs[i] ws[j] + bias[j]
//
// The sums are 32-bit integers: they are exact for K < 2^31 / 128^2 = 131072,
// so that splitting K over workgroups changes no bit of the result.

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include <algorithm>

#include "tile_product.h"

using namespace tile_product;

namespace {

template <class T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen(float v) { return v; }
template <> __device__ __forceinline__ float widen(_Float16 v) { return v; }
template <> __device__ __forceinline__ float widen(__bf16 v) {
  return (float)v;
}

// ---------------------------------------------------------------------------
// quantize
// ---------------------------------------------------------------------------

// rne(x / s) with the quotient taken exactly. x * (1 / s) is off by less than
// one step of q next to the middle of two integers only; the remainder
// x - q s is a multiple of s's last bit, so the fma gives it without a
// rounding and says on which side x lies.
__device__ __forceinline__ int nearest(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, s, x);
  const float a = fabsf(r), h = 0.5f * s;
  const bool odd = ((int)q) & 1;
  if (a > h || (a == h && odd)) q += copysignf(1.0f, r);
  return (int)q;
}

struct RowScale {
  float s, inv;
  bool fine, tiny;
  __device__ __forceinline__ RowScale(float big) {
    s = __fdiv_rn(big, 127.0f);
    fine = big < INFINITY;  // no infinity and no NaN
    tiny = s < 1e-36f;      // 1 / s or x - q s would leave the normal range
    inv = __fdiv_rn(1.0f, s);
  }
  __device__ __forceinline__ float scale() const { return fine ? s : NAN; }
  __device__ __forceinline__ int operator()(float x) const {
    if (!fine || s == 0.0f) return 0;
    if (tiny) {
      const double q = rint((double)x / (double)s);
      return (int)fmin(127.0, fmax(-127.0, q));
    }
    return nearest(x, s, inv);
  }
};

// NaN has to survive the maximum: fmaxf would drop it.
__device__ __forceinline__ float max_abs(float m, float x) {
  const float a = fabsf(x);
  return (a > m || a != a) ? a : m;
}

template <class T, int VEC> struct Chunk {
  struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[VEC]; };
};

// A row for LANES lanes, each holding CH chunks of 16 bytes of it between the
// two passes (maximum, then rounding), so that x is read once. Memory-bound:
// a few comparisons and about ten operations for the rounding of a value,
// against the 5 (or 3) bytes that it moves.
template <class T, int LANES, int CH>
__global__ __launch_bounds__(256) void quantize_rows_k(
    const T* __restrict__ x, long m, int k, long stride,
    int8_t* __restrict__ q, long qstride, float* __restrict__ scale) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int ROWS = 256 / LANES;
  typedef typename Chunk<T, VEC>::Raw Raw;
  __shared__ float part[4];
  const int lane = threadIdx.x % LANES;
  const long row = (long)blockIdx.x * ROWS + threadIdx.x / LANES;
  const bool here = row < m;
  const T* xr = x + (here ? row : 0) * stride;
  float v[CH][VEC];
  float big = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (c * LANES + lane) * VEC;
    if (at + VEC <= k) {
      const Raw raw = *(const Raw*)(xr + at);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[c][e] = widen(raw.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        v[c][e] = at + e < k ? widen(xr[at + e]) : 0.0f;
    }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < VEC; ++e) big = max_abs(big, v[c][e]);
#pragma unroll
  for (int d = 1; d < (LANES < 64 ? LANES : 64); d <<= 1)
    big = max_abs(big, __shfl_xor(big, d));
  if (LANES > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = big;
    __syncthreads();
    big = part[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) big = max_abs(big, part[w]);
  }
  if (!here) return;
  const RowScale rs(big);
  if (lane == 0) scale[row] = rs.scale();
  int8_t* qr = q + row * qstride;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (c * LANES + lane) * VEC;
    uint32_t w[VEC / 4];
#pragma unroll
    for (int d = 0; d < VEC / 4; ++d) {
      w[d] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[d] |= (uint32_t)(uint8_t)(int8_t)rs(v[c][4 * d + e]) << (8 * e);
    }
    // the row's last 16 bytes are filled up with zeros
    if (at < qstride) {
#pragma unroll
      for (int d = 0; d < VEC / 4; ++d) ((uint32_t*)(qr + at))[d] = w[d];
    }
  }
}

// Rows longer than the registers of a workgroup hold: read twice.
template <class T>
__global__ __launch_bounds__(256) void quantize_long_rows_k(
    const T* __restrict__ x, long m, long k, long stride,
    int8_t* __restrict__ q, long qstride, float* __restrict__ scale) {
  constexpr int VEC = 16 / sizeof(T);
  typedef typename Chunk<T, VEC>::Raw Raw;
  __shared__ float part[4];
  const long row = blockIdx.x;
  const T* xr = x + row * stride;
  float big = 0.0f;
  for (long at = (long)threadIdx.x * VEC; at < k; at += 256 * VEC) {
    if (at + VEC <= k) {
      const Raw raw = *(const Raw*)(xr + at);
#pragma unroll
      for (int e = 0; e < VEC; ++e) big = max_abs(big, widen(raw.v[e]));
    } else {
      for (long e = at; e < k; ++e) big = max_abs(big, widen(xr[e]));
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) big = max_abs(big, __shfl_xor(big, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = big;
  __syncthreads();
  big = part[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) big = max_abs(big, part[w]);
  const RowScale rs(big);
  if (threadIdx.x == 0) scale[row] = rs.scale();
  int8_t* qr = q + row * qstride;
  for (long at = (long)threadIdx.x * VEC; at < qstride; at += 256 * VEC) {
    uint32_t w[VEC / 4];
    if (at + VEC <= k) {
      const Raw raw = *(const Raw*)(xr + at);
#pragma unroll
      for (int d = 0; d < VEC / 4; ++d) {
        w[d] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[d] |= (uint32_t)(uint8_t)(int8_t)rs(widen(raw.v[4 * d + e]))
                  << (8 * e);
      }
    } else {
#pragma unroll
      for (int d = 0; d < VEC / 4; ++d) {
        w[d] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const long i = at + 4 * d + e;
          const int v = i < k ? rs(widen(xr[i])) : 0;
          w[d] |= (uint32_t)(uint8_t)(int8_t)v << (8 * e);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < VEC / 4; ++d) ((uint32_t*)(qr + at))[d] = w[d];
  }
}

template <class T, int LANES, int CH>
void quantize_as(const T* x, long m, long k, long stride, int8_t* q,
                 long qstride, float* scale, hipStream_t st) {
  const long rows = 256 / LANES;
  hipLaunchKernelGGL((quantize_rows_k<T, LANES, CH>),
                     dim3((unsigned)((m + rows - 1) / rows)), dim3(256), 0,
                     st, x, m, (int)k, stride, q, qstride, scale);
}

template <class T>
void quantize(const T* x, long m, long k, long stride, int8_t* q,
              long qstride, float* scale, hipStream_t st) {
  // chunks of the padded row, so that its zeros are written too
  const long chunks = (qstride * (long)sizeof(T) + 15) / 16;
  if (chunks <= 4) quantize_as<T, 4, 1>(x, m, k, stride, q, qstride, scale, st);
  else if (chunks <= 8) quantize_as<T, 8, 1>(x, m, k, stride, q, qstride, scale, st);
  else if (chunks <= 16) quantize_as<T, 16, 1>(x, m, k, stride, q, qstride, scale, st);
  else if (chunks <= 32) quantize_as<T, 32, 1>(x, m, k, stride, q, qstride, scale, st);
  else if (chunks <= 64) quantize_as<T, 64, 1>(x, m, k, stride, q, qstride, scale, st);
  else if (chunks <= 128) quantize_as<T, 64, 2>(x, m, k, stride, q, qstride, scale, st);
  else if (chunks <= 256) quantize_as<T, 256, 1>(x, m, k, stride, q, qstride, scale, st);
  else if (chunks <= 512) quantize_as<T, 256, 2>(x, m, k, stride, q, qstride, scale, st);
  else if (chunks <= 1024) quantize_as<T, 256, 4>(x, m, k, stride, q, qstride, scale, st);
  else if (chunks <= 2048) quantize_as<T, 256, 8>(x, m, k, stride, q, qstride, scale, st);
  else
    hipLaunchKernelGGL((quantize_long_rows_k<T>), dim3((unsigned)m),
                       dim3(256), 0, st, x, m, k, stride, q, qstride, scale);
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------

struct Scales {
  const float* xs;
  const float* ws;
  const float* bias;  // may be null
  void* out;
  long n;             // columns, and the output's row stride
  int vec;            // rows of the output begin at multiples of 4 values
};

template <class T> __device__ __forceinline__ T narrow(float v) {
  return (T)v;
}

// Four columns side by side of one row: y = acc xs ws + bias, rounded once.
template <class T>
__device__ __forceinline__ void store4(const Scales& e, long m, long n,
                                       const v4i& acc) {
  const float xs = e.xs[m];
  T* out = (T*)e.out + m * e.n + n;
  T v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < e.n)
      v[r] = narrow<T>(fmaf((float)acc[r] * xs, e.ws[n + r],
                            e.bias ? e.bias[n + r] : 0.0f));
  if (e.vec && n + 4 <= e.n) {
    struct __attribute__((aligned(4 * sizeof(T)))) Four { T v[4]; };
    *(Four*)out = Four{v[0], v[1], v[2], v[3]};
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < e.n) out[r] = v[r];
  }
}

// `slab` not null: the sums of this split of K, for joining later.
template <class T, int BM, int WM, int WN, int STAGES, int GROUPS>
__global__ __launch_bounds__(GROUPS * (BM / WM) * (BM / WN) * 64)
void int8_tile_k(
    Sources s, Scales e, int tm, int tn, int per, int* __restrict__ slab) {
  constexpr int BN = BM;
  typedef Tile<v4i, BM, BN, WM, WN, STAGES, GROUPS> P;
  __shared__ __attribute__((aligned(16))) char lds[P::kLds];
  int ti, tj;
  banded(xcd_contiguous(blockIdx.x, gridDim.x), tm, tn, ti, tj);
  const int steps = (s.kbytes + kStep - 1) / kStep;
  const int first = blockIdx.y * per, last = min(steps, first + per);
  v4i acc[P::MI][P::NJ];
  P::run(s, ti * BM, tj * BN, 0, first, last, lds, acc);
  int wm, wn;
  if (P::place(wm, wn)) return;
  const int lane = threadIdx.x & 63;
  const int m0 = ti * BM + wm + (lane & 15);
  const int n0 = tj * BN + wn + (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < P::MI; ++i) {
    const long m = m0 + i * 16;
    if (m >= s.rows_a) continue;
#pragma unroll
    for (int j = 0; j < P::NJ; ++j) {
      const long n = n0 + j * 16;
      if (n >= s.rows_b) continue;
      if (slab) {
        int* to = slab + ((long)blockIdx.y * s.rows_a + m) * s.rows_b + n;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < s.rows_b) to[r] = acc[i][j][r];
      } else {
        store4<T>(e, m, n, acc[i][j]);
      }
    }
  }
}

// Few rows of x (at most 16 MT): the weights' bytes are what counts. A wave
// takes 16 output channels straight from memory to registers, no LDS; the
// four waves of a workgroup, and gridDim.y workgroups, share out K.
template <class T, int MT>
__global__ __launch_bounds__(256) void int8_few_rows_k(
    Sources s, Scales e, int per, int* __restrict__ slab) {
  __shared__ v4i sums[4][MT][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16;
  const int chunk = lane >> 4;
  const int steps = (s.kbytes + kStep - 1) / kStep;
  const int tail = s.kbytes - (steps - 1) * kStep;
  const int first = blockIdx.y * per, last = min(steps, first + per);
  const char* pw = s.b[0] +
                   (long)min(n0 + (lane & 15), s.rows_b - 1) * s.row_b;
  const char* px[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    px[t] = s.a[0] +
            (long)min(t * 16 + (lane & 15), s.rows_a - 1) * s.row_a;
  v4i acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = v4i{0, 0, 0, 0};
  auto step = [&](int k, bool cut) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int c = (kk * 4 + chunk) * 16;
      const long at = (long)k * kStep + (cut && c >= tail ? 0 : c);
      v4i w = *(const v4i*)(pw + at);
      if (cut) w = keep_bytes(w, tail - c);
#pragma unroll
      for (int t = 0; t < MT; ++t)
        acc[t] = mma(w, *(const v4i*)(px[t] + at), acc[t]);
    }
  };
  const bool mine = last == steps && tail < kStep;  // the cut step is here
  const int whole = mine ? last - 1 : last;
  int k = first + wave;
  for (; k + 12 < whole; k += 16) {
#pragma unroll
    for (int u = 0; u < 4; ++u) step(k + 4 * u, false);
  }
  for (; k < whole; k += 4) step(k, false);
  if (mine && k == last - 1) step(k, true);
#pragma unroll
  for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < MT; t += 4) {
    v4i v = sums[0][t][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) v += sums[w][t][lane];
    const long m = t * 16 + (lane & 15), n = n0 + chunk * 4;
    if (m >= s.rows_a || n >= s.rows_b) continue;
    if (slab) {
      int* to = slab + ((long)blockIdx.y * s.rows_a + m) * s.rows_b + n;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < s.rows_b) to[r] = v[r];
    } else {
      store4<T>(e, m, n, v);
    }
  }
}

template <class T>
__global__ __launch_bounds__(256) void int8_join_k(
    const int* __restrict__ slab, int splits, long m, Scales e) {
  const long total = m * e.n;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  int sum = 0;
  for (int p = 0; p < splits; ++p) sum += slab[p * total + i];
  const long row = i / e.n, n = i - row * e.n;
  ((T*)e.out)[i] = narrow<T>(fmaf((float)sum * e.xs[row], e.ws[n],
                                  e.bias ? e.bias[n] : 0.0f));
}

// How a product is computed: by `rows` (16, 32 or 64) rows without LDS, or in
// square tiles of `size`, each with K in `splits` parts of `per` steps.
struct Plan { int rows, size, tm, tn, splits, per; };

Plan plan_of(long m, long n, long k) {
  Plan p = {};
  const int steps = (int)((k + kStep - 1) / kStep);
  if (m <= 64) {
    // enough workgroups for two on each CU, of 16 steps at least
    p.rows = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    p.tm = 1;
    p.tn = (int)((n + 15) / 16);
    long want = p.tn >= 512 ? 1 : (512 + p.tn - 1) / p.tn;
    want = std::min(want, std::min(64L, std::max(1L, (long)steps / 16)));
    p.per = (int)((steps + want - 1) / want);
  } else {
    // the tile and the split that need the least time; joining the parts
    // takes a launch, and writes and reads them at 4 TB/s
    double best = 1e30;
    for (const TileCost& c : kTiles)
      for (int splits = 1; splits <= 64 && splits * 4 <= steps + 3;
           splits *= 2) {
        const long tm = (m + c.size - 1) / c.size;
        const long tn = (n + c.size - 1) / c.size;
        const int per = (steps + splits - 1) / splits;
        const double join =
            splits > 1 ? 4.0 + 8e-6 * splits * m * n / 4.0 : 0.0;
        const double t = per * step_time(c, tm * tn * splits) + join;
        if (t < best) {
          best = t;
          p.size = c.size;
          p.tm = (int)tm;
          p.tn = (int)tn;
          p.per = per;
        }
      }
  }
  p.splits = (steps + p.per - 1) / p.per;
  return p;
}

template <class T>
void product(const Sources& s, const Scales& e, const Plan& p, int* slab,
             hipStream_t st) {
  const dim3 grid(p.tm * p.tn, p.splits);
#define FEW(MT)                                                           \
  hipLaunchKernelGGL((int8_few_rows_k<T, MT>), grid, dim3(256), 0, st, s, \
                     e, p.per, slab)
#define TILE(BM, WM, WN, STAGES, GROUPS)                                 \
  hipLaunchKernelGGL((int8_tile_k<T, BM, WM, WN, STAGES, GROUPS>), grid, \
                     dim3(GROUPS * (BM / WM) * (BM / WN) * 64), 0, st,   \
                     s, e, p.tm, p.tn, p.per, slab)
  if (p.rows == 16) FEW(1);
  else if (p.rows == 32) FEW(2);
  else if (p.rows == 64) FEW(4);
  else {
    const bool alone = (long)p.tm * p.tn * p.splits <= 256;
    BY_TILE_SIZE(p.size, alone, TILE)
  }
#undef FEW
#undef TILE
  if (slab) {
    const long total = (long)s.rows_a * e.n;
    hipLaunchKernelGGL((int8_join_k<T>), dim3((unsigned)((total + 255) / 256)),
                       dim3(256), 0, st, slab, p.splits, (long)s.rows_a, e);
  }
}

}  // namespace

// dtype: 0 float32, 1 float16, 2 bfloat16.
extern "C" void launch_quantize_rows(const void* x, int dtype, long m, long k,
                                     long stride, int8_t* q, long qstride,
                                     float* scale, hipStream_t st) {
  if (dtype == 0)
    quantize((const float*)x, m, k, stride, q, qstride, scale, st);
  else if (dtype == 1)
    quantize((const _Float16*)x, m, k, stride, q, qstride, scale, st);
  else
    quantize((const __bf16*)x, m, k, stride, q, qstride, scale, st);
}

// Values of the 32-bit workspace that the product needs (0: none).
extern "C" long int8_product_workspace(long m, long n, long k) {
  const Plan p = plan_of(m, n, k);
  return p.splits > 1 ? p.splits * m * n : 0;
}

extern "C" void launch_int8_product(const int8_t* xq, long xstride,
                                    const float* xs, const int8_t* wq,
                                    long wstride, const float* ws,
                                    const float* bias, long m, long n, long k,
                                    void* out, int dtype, int* work,
                                    hipStream_t st) {
  const Plan p = plan_of(m, n, k);
  Sources s = {};
  s.a[0] = (const char*)xq;
  s.b[0] = (const char*)wq;
  s.row_a = (unsigned)xstride;
  s.row_b = (unsigned)wstride;
  s.rows_a = (int)m;
  s.rows_b = (int)n;
  s.kbytes = (int)k;
  s.parts = 1;
  Scales e = {xs, ws, bias, out, n, n % 4 == 0};
  int* slab = p.splits > 1 ? work : nullptr;
  if (dtype == 0)
    product<float>(s, e, p, slab, st);
  else if (dtype == 1)
    product<_Float16>(s, e, p, slab, st);
  else
    product<__bf16>(s, e, p, slab, st);
}
