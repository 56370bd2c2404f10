// The main loop of the matrix products C = A B^T, with both operands' rows
// contiguous along the summed axis ("K"). It counts K in bytes: a lane of
// v_mfma_i32_16x16x64_i8 and one of v_mfma_f32_16x16x32_f16 take 16 bytes of
// a row each, from the same places, so that one loader, one LDS layout and
// one loop serve both types.
//
// A workgroup computes a BM x BN tile in steps of 128 bytes of K. The step's
// rows go to LDS by DMA (global_load_lds, 16 bytes a lane), which writes
// lanes in order; the XOR swizzle that keeps ds_read_b128 free of bank
// conflicts (chunk c of row r sits in place c ^ (r & 7)) is therefore put
// into the address that each lane reads from.
#pragma once
#include <hip/hip_runtime.h>

namespace tile_product {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kStep = 128;  // bytes of K in one step

// What a launch reads. `parts` pairs of operands are summed as if their K
// were joined (a value split in two 16-bit halves takes two or three).
struct Sources {
  const char* a[3];
  const char* b[3];
  long batch_a, batch_b;   // bytes from one batch entry to the next
  unsigned row_a, row_b;   // bytes from row to row: a multiple of 16
  int rows_a, rows_b;
  int kbytes;              // bytes of a row that count
  int parts;
};

// Workgroups go round the 8 XCDs in turn. This gives each XCD a contiguous
// run of tiles, whose rows its own L2 then holds.
__device__ __forceinline__ int xcd_contiguous(int b, int n) {
  const int q = n >> 3, r = n & 7;
  const int x = b & 7;
  return x * q + min(x, r) + (b >> 3);
}

// Tile t of a grid of tm x tn, in bands of 8 rows of tiles, so that tiles
// that run at the same time share rows of both operands.
__device__ __forceinline__ void banded(int t, int tm, int tn, int& i, int& j) {
  const int band = t / (8 * tn);
  const int first = band * 8;
  const int high = min(8, tm - first);
  const int in = t - first * tn;
  i = first + in % high;
  j = in / high;
}

// Tile t of the lower triangle (i >= j), row by row.
__device__ __forceinline__ void triangle(int t, int& i, int& j) {
  i = (int)((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
  while ((i + 1) * (i + 2) / 2 <= t) ++i;
  while (i * (i + 1) / 2 > t) --i;
  j = t - i * (i + 1) / 2;
}

// The bytes of a 16-byte chunk behind the first `valid` made zero.
__device__ __forceinline__ v4i keep_bytes(v4i v, int valid) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int n = valid - 4 * d;
    const unsigned m = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
    v[d] &= (int)m;
  }
  return v;
}

__device__ __forceinline__ v4i mma(v4i x, v4i y, v4i c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(x, y, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mma(v4i x, v4i y, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0, 0);
}

// BM x BN: the workgroup's tile, WM x WN: a wave's. ACC is v4i for 8-bit
// integers and v4f for 16-bit floats.
template <class ACC, int BM, int BN, int WM, int WN>
struct Tile {
  static constexpr int kWaves = (BM / WM) * (BN / WN);
  static constexpr int kThreads = kWaves * 64;
  static constexpr int MI = WM / 16, NJ = WN / 16;
  static constexpr int kStage = (BM + BN) * kStep;
  static constexpr int kLds = 2 * kStage;
  static constexpr bool kInt = __is_same(ACC, v4i);

  // acc[i][j][r] is the sum for row  m = i * 16 + lane % 16  and column
  // n = j * 16 + lane / 16 * 4 + r  of the wave's part of the tile: B goes in
  // as the first operand, so that a lane ends with four columns side by side.
  static __device__ __forceinline__ void run(const Sources& s, int m0, int n0,
                                             long batch, int first, int last,
                                             char* lds,
                                             ACC (&acc)[MI][NJ]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / (BN / WN), wn = wave % (BN / WN);
    constexpr int LA = BM / 8 / kWaves, LB = BN / 8 / kWaves;
    const int r8 = lane >> 3;
    const int c16 = ((lane & 7) ^ r8) * 16;
    // rows behind the last are read from the last one; nothing is stored
    // from what they give
    unsigned oa[LA], ob[LB];
#pragma unroll
    for (int i = 0; i < LA; ++i)
      oa[i] = (unsigned)(min(m0 + (i * kWaves + wave) * 8 + r8,
                             s.rows_a - 1) - m0) * s.row_a;
#pragma unroll
    for (int i = 0; i < LB; ++i)
      ob[i] = (unsigned)(min(n0 + (i * kWaves + wave) * 8 + r8,
                             s.rows_b - 1) - n0) * s.row_b;
    const int steps = (s.kbytes + kStep - 1) / kStep;
    const int tail = s.kbytes - (steps - 1) * kStep;  // bytes of the last step
    const long at_a = batch * s.batch_a + (long)m0 * s.row_a;
    const long at_b = batch * s.batch_b + (long)n0 * s.row_b;

    auto load = [&](int t, int buf) {
      const int part = t / steps, k = t - part * steps;
      const char* pa = s.a[part] + at_a + (long)k * kStep;
      const char* pb = s.b[part] + at_b + (long)k * kStep;
      // a chunk that begins behind the row's end is read from the step's
      // first one instead, and masked below
      const unsigned c = (k == steps - 1 && c16 >= tail) ? 0 : c16;
      char* la = lds + buf * kStage + wave * 1024;
      char* lb = la + BM * kStep;
#pragma unroll
      for (int i = 0; i < LA; ++i)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(pa + (oa[i] + c)),
            (__attribute__((address_space(3))) void*)(la + i * kWaves * 1024),
            16, 0, 0);
#pragma unroll
      for (int i = 0; i < LB; ++i)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(pb + (ob[i] + c)),
            (__attribute__((address_space(3))) void*)(lb + i * kWaves * 1024),
            16, 0, 0);
    };

#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = ACC{0, 0, 0, 0};

    const int row = (lane & 15) * kStep;
    load(first, 0);
    for (int t = first; t < last; ++t) {
      const int buf = (t - first) & 1;
      // one barrier a step: the loads of this step are in, and every wave
      // has read the other buffer
      __syncthreads();
      if (t + 1 < last) load(t + 1, buf ^ 1);
      const char* la = lds + buf * kStage + wm * WM * kStep + row;
      const char* lb = lds + buf * kStage + (BM + wn * WN) * kStep + row;
      const bool cut = kInt && tail < kStep && t % steps == steps - 1;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int chunk = kk * 4 + (lane >> 4);
        const int place = (chunk ^ (lane & 7)) * 16;
        v4i fa[MI], fb[NJ];
#pragma unroll
        for (int i = 0; i < MI; ++i)
          fa[i] = *(const v4i*)(la + i * 16 * kStep + place);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          fb[j] = *(const v4i*)(lb + j * 16 * kStep + place);
        if (cut)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            fb[j] = keep_bytes(fb[j], tail - chunk * 16);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
      }
    }
    __syncthreads();
  }
};

}  // namespace tile_product
