// Rows into 8-bit floating point (fp8.h holds the format), plain or behind a gated unit: x [M, K] -> codes [M, 128 U] and scale bytes
// [M, 4 U4], or x [M, 2 K] (gate columns, then up columns) -> those of act(g) u rounded to x's type.
//
// Bound: a pass over memory (2 or 4 bytes in, 1 out).  16 neighbouring lanes hold a block of 128, eight values each: its largest
// magnitude is found by register moves, nothing is read twice and nothing is kept.  8,192 x 5,120 bfloat16: 25 us, 5.0 TB/s, what a copy
// reaches; a row of 5,120: the launch.
#include "fp8.h"

// Eight values of a block whose others 15 neighbouring lanes hold: their codes, and the block's byte.
__device__ __forceinline__ int eight_codes(const float (&v)[8], uint32_t (&c)[2]) {
  uint32_t top = 0;
  bool bad[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t m = __float_as_uint(v[i]) & 0x7fffffffu;
    bad[i] = m >= 0x7f800000u;
    if (!bad[i] && m > top) top = m;
  }
  float t = __uint_as_float(top);
  t = fmaxf(t, row_rotated<8>(t));
  t = fmaxf(t, row_rotated<4>(t));
  t = fmaxf(t, row_rotated<2>(t));
  t = fmaxf(t, row_rotated<1>(t));
  const int s = f8_scale_of(__float_as_uint(t));
  const float scale = f8_scale_value(s);
  c[0] = f8_codes4(v[0], v[1], v[2], v[3], scale);
  c[1] = f8_codes4(v[4], v[5], v[6], v[7], scale);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (bad[i]) c[i / 4] = (c[i / 4] & ~(0xffu << (i % 4 * 8))) | kF8Nan << (i % 4 * 8);
  return s;
}

// Eight values from a row's k on (zeros behind its K), in loads of 16 bytes at whatever address: the memory takes any.
template <typename T> __device__ __forceinline__ void load_eight(const T* __restrict__ row, int k, int K, float (&v)[8]) {
  if (k + 8 <= K) {
    T t[8];
    __builtin_memcpy(t, row + k, sizeof(t));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f32(row[k + i]) : 0.f;
  }
}

template <typename T, bool GATED>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                       long long n_blocks, int K, int U, int su, GatedAct act) {
  const long long b = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * 16 + (threadIdx.x >> 4);
  if (b >= n_blocks) return;                   // (16 lanes at once)
  const int l = threadIdx.x & 15;
  const long long row = b / U;
  const int u = (int)(b - row * U), k = u * kF8Block + l * 8;
  const T* src = x + row * (GATED ? 2 * (long long)K : K);
  float v[8];
  load_eight(src, k, K, v);
  if constexpr (GATED) {
    float w[8];
    load_eight(src + K, k, K, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(from_f32<T>(gated_f32(act, v[i], w[i], 1.f, false)));
  }
  uint32_t c[2];
  const int s = eight_codes(v, c);
  *reinterpret_cast<uint2*>(codes + b * kF8Block + l * 8) = make_uint2(c[0], c[1]);
  if (l == 0) scales[row * su + u] = (uint8_t)s;
  else if (u == U - 1 && U - 1 + l < su) scales[row * su + U - 1 + l] = 127;      // (the bytes behind the last block: a scale of one)
}

// dtype of x (DT_*); act 0: x [M, K]; else the gated unit's code, x [M, 2K].
SHARPI_EXPORT int sharpi_fp8_rows(const void* x, int dtype, void* codes, void* scales, int M, int K, int act, float limit, hipStream_t stream) {
  if (M <= 0) return SHARPI_OK;
  const GatedAct ga{act, limit};
  if (K <= 0 || K >= kF8MostK || act < 0 || (act > 0 && !act_known(ga))) return SHARPI_ERR_ARG;
  const int U = f8_blocks(K), su = f8_scale_stride(K);
  const long long n = (long long)M * U;
  const long long blocks = (n + 15) / 16, across = blocks < 1 << 20 ? blocks : 1 << 20;      // (a launch has at most 2^32 threads along x)
  if ((blocks + across - 1) / across > 0xffff) return SHARPI_ERR_ARG;
  const dim3 grid((unsigned)across, (unsigned)((blocks + across - 1) / across)), block(256);
#define FR(T, G) fp8_rows_kernel<T, G><<<grid, block, 0, stream>>>((const T*)x, (uint8_t*)codes, (uint8_t*)scales, n, K, U, su, ga)
  if (dtype == DT_BF16) { if (act) FR(bf16_t, true); else FR(bf16_t, false); }
  else if (dtype == DT_F32) { if (act) FR(float, true); else FR(float, false); }
  else return SHARPI_ERR_ARG;
#undef FR
  SHARPI_CHECK_LAUNCH();
  return SHARPI_OK;
}

// Matrices [N, K] (GATED: gate rows, then as many up rows) into the stored order of tiles, each in one pass.  16 lanes hold a block of 128 as above; a block
// of threads takes 16 rows of a tile, so that a run of 256 bytes of the stored order is written at a time.  Bound: a pass over memory; run when a
// program loads its weights.
template <typename T>
__global__ __launch_bounds__(256) void fp8_weight_kernel(const T* __restrict__ w, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int N, int K, int U,
                                                         int stored, int gated) {
  const int l = threadIdx.x & 15, U4 = (U + 3) >> 2, half = blockIdx.x & 1;
  const int u = (blockIdx.x >> 1) % U, tile = (blockIdx.x >> 1) / U, r = half * 16 + (threadIdx.x >> 4);
  const size_t e = blockIdx.y, at = e * (stored / kF8Tile) + tile;
  // the row of the matrix that is stored there (each half of a gated one is filled up by itself), if one is
  const int part = gated ? stored / 2 : stored, mine = gated ? N / 2 : N, row = tile * kF8Tile + r, in = row % part;
  const bool real = in < mine;
  const T* src = w + (e * N + (row / part) * mine + in) * K;
  const int k = u * kF8Block + l * 8;
  float v[8];
  load_eight(src, real ? k : K, K, v);
  uint32_t c[2];
  const int s = eight_codes(v, c);
  // k = 64 s + 32 g + 16 p + byte: lane l has byte 8 (l & 1) of piece l / 2 % 2 of group l / 4 % 2 of half l / 8
  uint8_t* to = codes + (at * U + u) * kF8TileBytes + (l >> 3) * 2048 + (l >> 1 & 1) * 1024 + (l >> 2 & 1) * 512 + r * 16 + (l & 1) * 8;
  *reinterpret_cast<uint2*>(to) = make_uint2(c[0], c[1]);
  uint8_t* byte = scales + (at * U4 + (u >> 2)) * 128 + r * 4;
  if (l == 0) byte[u & 3] = real ? (uint8_t)s : 127;
  else if (u == U - 1 && (u & 3) + l < 4) byte[(u & 3) + l] = 127;
}

// codes, scales: of `matrices` of them, each of f8_padded_rows(N) stored rows (gated: twice those of N / 2).
SHARPI_EXPORT int sharpi_fp8_weight(const void* w, int dtype, void* codes, void* scales, int matrices, int N, int K, int gated, hipStream_t stream) {
  if (matrices <= 0) return SHARPI_OK;
  if (N <= 0 || K <= 0 || K >= kF8MostK || (gated && N % 2) || matrices > 0xffff) return SHARPI_ERR_ARG;
  const int U = f8_blocks(K), stored = gated ? 2 * f8_padded_rows(N / 2) : f8_padded_rows(N);
  const long long blocks = (long long)stored / kF8Tile * U * 2;
  if (blocks > 0xffffff) return SHARPI_ERR_ARG;             // (of 256 threads each, of which a launch has at most 2^32 along x)
  const dim3 grid((unsigned)blocks, (unsigned)matrices), block(256);
#define FW(T) fp8_weight_kernel<T><<<grid, block, 0, stream>>>((const T*)w, (uint8_t*)codes, (uint8_t*)scales, N, K, U, stored, gated)
  if (dtype == DT_BF16) FW(bf16_t);
  else if (dtype == DT_F32) FW(float);
  else return SHARPI_ERR_ARG;
#undef FW
  SHARPI_CHECK_LAUNCH();
  return SHARPI_OK;
}

// out[t] = sum_j w[t, j] y[inv_pos[t, j]] (+ shared[t]) of float rows, rounded to bfloat16 once; picks outside 0 .. n_experts - 1 have no row and add nothing.
// Bound: a pass over the rows (4,096 rows of 5,120 into 2,048: 105 MB in 21 us with the launch).
template <bool WIDE>
__global__ __launch_bounds__(256) void fp8_combine_kernel(const float* __restrict__ y, const int* __restrict__ inv_pos, const int* __restrict__ ids,
                                                          const float* __restrict__ shared, const float* __restrict__ w, bf16_t* __restrict__ out,
                                                          int columns, int k, int n_experts) {
  constexpr int V = WIDE ? 8 : 1;
  const size_t t = blockIdx.x;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (c >= columns) return;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  auto add = [&](const float* row, float weight) {
    float v[V];
    if constexpr (WIDE) load8(row + c, v);
    else v[0] = row[c];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = fmaf(weight, v[i], acc[i]);
  };
  for (int j = 0; j < k; ++j) {
    const size_t p = t * k + j;
    if ((unsigned)ids[p] < (unsigned)n_experts) add(y + (size_t)inv_pos[p] * columns, w ? w[p] : 1.f);
  }
  if (shared) add(shared + t * columns, 1.f);
  if constexpr (WIDE) store8(out + t * columns + c, acc);
  else out[t * columns + c] = f32_to_bf16(acc[0]);
}

SHARPI_EXPORT int sharpi_fp8_combine(const float* y, const int* inv_pos, const int* ids, const float* shared, const float* w, void* out, int n_tokens,
                                     int columns, int k, int n_experts, hipStream_t stream) {
  if (n_tokens <= 0) return SHARPI_OK;
  if (columns <= 0 || k <= 0 || n_tokens > 0xffffff || columns > kF8MostK - 256) return SHARPI_ERR_ARG;
  const bool wide = columns % 8 == 0 && (((uintptr_t)y | (uintptr_t)out | (uintptr_t)shared) & 15) == 0;
  const dim3 grid((unsigned)n_tokens, (unsigned)ceil_div(columns, wide ? 2048 : 256)), block(256);
  if (wide) fp8_combine_kernel<true><<<grid, block, 0, stream>>>(y, inv_pos, ids, shared, w, (bf16_t*)out, columns, k, n_experts);
  else fp8_combine_kernel<false><<<grid, block, 0, stream>>>(y, inv_pos, ids, shared, w, (bf16_t*)out, columns, k, n_experts);
  SHARPI_CHECK_LAUNCH();
  return SHARPI_OK;
}

// out = the sum of `shares` arrays of n floats on end, in their order, rounded to bfloat16.  Bound: a pass over them.
__global__ __launch_bounds__(256) void fp8_join_kernel(const float* __restrict__ part, bf16_t* __restrict__ out, long long n, int shares) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  if ((n & 3) == 0 && (((uintptr_t)part | (uintptr_t)out) & 15) == 0) {
    f32x4 v = *reinterpret_cast<const f32x4*>(part + i);
    for (int s = 1; s < shares; ++s) v += *reinterpret_cast<const f32x4*>(part + s * n + i);
    *reinterpret_cast<uint2*>(out + i) = make_uint2(f32_to_bf16_pair(v[0], v[1]), f32_to_bf16_pair(v[2], v[3]));
    return;
  }
  for (int j = 0; j < 4 && i + j < n; ++j) {
    float v = part[i + j];
    for (int s = 1; s < shares; ++s) v += part[s * n + i + j];
    out[i + j] = f32_to_bf16(v);
  }
}

SHARPI_EXPORT int sharpi_fp8_join(const float* part, void* out, long long n, int shares, hipStream_t stream) {
  if (n <= 0) return SHARPI_OK;
  if (shares < 1 || (n + 1023) / 1024 > 0xffffff) return SHARPI_ERR_ARG;
  fp8_join_kernel<<<dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, stream>>>(part, (bf16_t*)out, n, shares);
  SHARPI_CHECK_LAUNCH();
  return SHARPI_OK;
}
