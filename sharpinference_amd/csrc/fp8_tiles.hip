// Products of many rows with weights in 8-bit floating point (fp8.h holds the format), in tiles on the scaled matrix instruction: one matrix, or
// the experts of a routing's sorted row list.  Two forms:
//   plain   out[row, :] = rows[row] W_e^T, bfloat16
//   gated   act(s g) (s u) with (g | u) the product, rounded to bfloat16 and quantised again: codes and scale bytes of the rows that the
//           second half of a feed-forward reads.  A block's 128 output columns are one block of the format, so the epilogue has what
//           it needs, and neither (g | u) nor the unquantised rows go to memory.
// Every output is one chain over k in ascending order: a row's result does not depend on which rows share its tile.
#include "fp8.h"

namespace {

constexpr int TW = 8;                  // waves a block: 2 along the rows x 4 along the columns
constexpr int TWC = 4;
constexpr int kTileCols = 256;         // weight rows of a block: 64 a column wave, two tiles of 32
constexpr int kMaxGroups = 1024;

struct F8Tiles {
  const uint8_t* x;          // codes [x_rows, 128 U]
  const uint8_t* xs;         // [x_rows, 4 U4]
  const uint8_t* w;          // [groups][w_rows / 32][U][4096]
  const uint8_t* ws;
  int U, w_rows;             // blocks of k; stored rows of one matrix
  const int* a_rows;         // [rows] or null
  const int* offsets;        // [groups + 1] or null (one group of `rows` rows)
  int rows, groups;          // rows of the sorted list at most
  int along;                 // rows behind these that one more matrix takes, in the order of x (0: none)
  int tiles, nb;             // row tiles in all at most; column blocks
};

// plain: out [rows, n_out].  gated: codes [rows, 128 f8_blocks(n_out)], scales [rows, f8_scale_stride(n_out)], score [rows] or null.
struct F8Out {
  bf16_t* out;
  uint8_t* codes;
  uint8_t* scales;
  const float* score;
  int n_out;
};

// MT: groups of 32 rows a wave; a tile has 64 MT rows.
template <int MT, bool GATED>
__global__ __launch_bounds__(TW* kWave) void fp8_tiles_kernel(F8Tiles p, F8Out o, GatedAct act) {
  constexpr int TM = 64 * MT;
  __shared__ int s_offset[kMaxGroups + 1];
  __shared__ int s_group, s_row0, s_end;
  __shared__ float s_top[TWC][GATED ? TM : 1];
  const int lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, g = lane >> 5;
  const int wr = wid / TWC, wc = wid % TWC;
  const int tile = blockIdx.x % p.tiles, nblock = blockIdx.x / p.tiles;
  int e = 0, row0 = tile * TM, row_end = min(p.rows, row0 + TM);
  if (p.offsets) {
    for (int i = threadIdx.x; i <= p.groups; i += TW * kWave) s_offset[i] = p.offsets[i];
    if (threadIdx.x == 0) s_group = -1;
    __syncthreads();
    if (wid == 0) {
      int before = 0;
      for (int c = 0; c < p.groups + (p.along > 0); c += kWave) {
        const int i = c + lane;
        const int from = i < p.groups ? s_offset[i] : p.rows, to = i < p.groups ? s_offset[i + 1] : i == p.groups ? p.rows + p.along : p.rows;
        const int mine = (to - from + TM - 1) / TM;
        int upto = mine;
#pragma unroll
        for (int k = 1; k < kWave; k <<= 1) {
          const int up = __shfl_up(upto, k, kWave);
          if (lane >= k) upto += up;
        }
        const int first = before + upto - mine;
        if (mine > 0 && tile >= first && tile < first + mine) {
          s_group = i;
          s_row0 = from + (tile - first) * TM;
          s_end = min(to, s_row0 + TM);
        }
        before += __shfl(upto, kWave - 1, kWave);
      }
    }
    __syncthreads();
    if (s_group < 0) return;
    e = __builtin_amdgcn_readfirstlane(s_group);
    row0 = __builtin_amdgcn_readfirstlane(s_row0);
    row_end = __builtin_amdgcn_readfirstlane(s_end);
  }
  const bool sorted = row0 < p.rows;             // of the sorted list, not of the rows behind it
  const int U4 = (p.U + 3) >> 2;
  // the wave's two weight tiles
  const int half = p.w_rows / 64;                // gated: tiles of the gate rows
  int wt[2];
  bool exists = true;
  if constexpr (GATED) {
    wt[0] = nblock * (kTileCols / 64) + wc;
    exists = wt[0] < half;
    wt[0] = min(wt[0], half - 1);
    wt[1] = wt[0] + half;
  } else {
#pragma unroll
    for (int t = 0; t < 2; ++t) wt[t] = min(nblock * (kTileCols / 32) + wc * 2 + t, p.w_rows / 32 - 1);
  }
  const uint8_t *wp[2], *wsp[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const size_t at = (size_t)e * (p.w_rows / 32) + wt[t];
    wp[t] = p.w + at * p.U * kF8TileBytes + lane * 16;
    wsp[t] = p.ws + at * U4 * 128 + r * 4;
  }
  const uint8_t *xp[MT], *xsp[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = min(row0 + (wr * MT + m) * 32 + r, row_end - 1);
    const size_t at = !p.a_rows ? row : sorted ? p.a_rows[row] : row - p.rows;
    xp[m] = p.x + at * p.U * kF8Block + g * 32;
    xsp[m] = p.xs + at * (U4 * 4);
  }
  f32x16 acc[2][MT];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][m][i] = 0.f;
  for (int u = 0; u < p.U; ++u) {
    int wb[2], xb[MT];
#pragma unroll
    for (int t = 0; t < 2; ++t) wb[t] = wsp[t][(u >> 2) * 128 + (u & 3)];
#pragma unroll
    for (int m = 0; m < MT; ++m) xb[m] = xsp[m][u];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      i32x8 wf[2], xf[MT];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const i32x4 a = *reinterpret_cast<const i32x4*>(wp[t] + (size_t)u * kF8TileBytes + s * 2048);
        const i32x4 b = *reinterpret_cast<const i32x4*>(wp[t] + (size_t)u * kF8TileBytes + s * 2048 + 1024);
        wf[t] = i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const i32x4 a = *reinterpret_cast<const i32x4*>(xp[m] + (size_t)u * kF8Block + s * 64);
        const i32x4 b = *reinterpret_cast<const i32x4*>(xp[m] + (size_t)u * kF8Block + s * 64 + 16);
        xf[m] = i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[t][m] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[t], xf[m], acc[t][m], 0, 0, 0, wb[t], 0, xb[m]);
    }
  }
  // a lane holds, of row row0 + (wr MT + m) 32 + r, columns 8 q + 4 g + 0..3 (q 0..3) of tile t
  if constexpr (!GATED) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = row0 + (wr * MT + m) * 32 + r;
      if (row >= row_end) continue;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = nblock * kTileCols + wc * 64 + t * 32 + q * 8 + g * 4;
          bf16_t* dst = o.out + (size_t)row * o.n_out + n;
          if (n + 4 <= o.n_out && ((uintptr_t)dst & 7) == 0) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(f32_to_bf16_pair(acc[t][m][4 * q], acc[t][m][4 * q + 1]),
                                                        f32_to_bf16_pair(acc[t][m][4 * q + 2], acc[t][m][4 * q + 3]));
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n + i < o.n_out) dst[i] = f32_to_bf16(acc[t][m][4 * q + i]);
          }
        }
    }
  } else {
    const int U2 = f8_blocks(o.n_out), su2 = f8_scale_stride(o.n_out);
    float h[MT][16];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int lrow = (wr * MT + m) * 32 + r, row = min(row0 + lrow, row_end - 1);
      const bool scaled = o.score != nullptr && sorted;
      const float sc = scaled ? o.score[row] : 1.f;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = exists ? bf16_to_f32(f32_to_bf16(gated_f32(act, acc[0][m][i], acc[1][m][i], sc, scaled))) : 0.f;
        const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
        if (b < 0x7f800000u && b > top) top = b;
        h[m][i] = v;
      }
      const float t2 = reduce32(__uint_as_float(top), MaxOf{});
      if (g == 0) s_top[wc][lrow] = t2;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int lrow = (wr * MT + m) * 32 + r, row = row0 + lrow;
      const float t = fmaxf(fmaxf(s_top[0][lrow], s_top[1][lrow]), fmaxf(s_top[2][lrow], s_top[3][lrow]));
      const int s = f8_scale_of(__float_as_uint(t));
      const float scale = f8_scale_value(s);
      if (row >= row_end) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t c = f8_codes4(h[m][4 * q], h[m][4 * q + 1], h[m][4 * q + 2], h[m][4 * q + 3], scale);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((__float_as_uint(h[m][4 * q + i]) & 0x7f800000u) == 0x7f800000u) c |= kF8Nan << (8 * i);
        *reinterpret_cast<uint32_t*>(o.codes + ((size_t)row * U2 + nblock) * kF8Block + wc * 32 + q * 8 + g * 4) = c;
      }
      if (wc == 0 && g == 0) o.scales[(size_t)row * su2 + nblock] = (uint8_t)s;
    }
  }
}

bool tiles_ok(const F8Tiles& p, int x_rows) {
  return p.rows > 0 && x_rows > 0 && p.U > 0 && p.w_rows > 0 && p.w_rows % kF8Tile == 0 && p.groups > 0 && p.groups < kMaxGroups && p.along >= 0 && (p.offsets || !p.along) && (long long)p.rows + p.along <= 0x7fffffffLL &&
         (long long)p.w_rows * p.U < 0x7fffffffLL && !(((uintptr_t)p.x | (uintptr_t)p.w) & 15) && (p.offsets || p.groups == 1);
}

template <bool GATED> int launch_tiles(F8Tiles p, const F8Out& o, GatedAct act, int height, hipStream_t stream) {
  const long long tiles = p.offsets ? (long long)p.rows / height + (p.rows < p.groups ? p.rows : p.groups) + (p.along + height - 1) / height
                                    : (p.rows + height - 1) / height;
  p.nb = ceil_div(o.n_out, GATED ? kTileCols / 2 : kTileCols);
  p.tiles = (int)tiles;
  if (tiles * p.nb > 0x7fffffffLL) return SHARPI_ERR_ARG;
  const dim3 grid((unsigned)(tiles * p.nb)), block(TW * kWave);
#define FT(MTV) fp8_tiles_kernel<MTV, GATED><<<grid, block, 0, stream>>>(p, o, act)
  if (height == 64) FT(1);
  else if (height == 128) FT(2);
  else if (height == 256) FT(4);
  else return SHARPI_ERR_ARG;
#undef FT
  SHARPI_CHECK_LAUNCH();
  return SHARPI_OK;
}

}  // namespace

// out [rows, N] bfloat16.  x: codes [x_rows, 128 U] and scales; w_rows: stored rows of one matrix; a_rows, offsets: of a sorted row list, or null; along: rows
// behind the list's `rows`, which matrix `groups` takes (row i reads row i - rows of x if there is a_rows); height: rows of a tile (64, 128, 256).
SHARPI_EXPORT int sharpi_fp8_tiles(const void* x, const void* x_scales, int x_rows, const void* w_codes, const void* w_scales, int w_rows, void* out,
                                   int rows, int N, int K, const int* a_rows, const int* offsets, int groups, int along, int height, hipStream_t stream) {
  if (rows <= 0) return SHARPI_OK;
  if (N <= 0 || K <= 0 || w_rows != f8_padded_rows(N)) return SHARPI_ERR_ARG;
  const F8Tiles p{(const uint8_t*)x, (const uint8_t*)x_scales, (const uint8_t*)w_codes, (const uint8_t*)w_scales, f8_blocks(K), w_rows, a_rows, offsets, rows, groups, along, 0, 0};
  if (!tiles_ok(p, x_rows)) return SHARPI_ERR_ARG;
  return launch_tiles<false>(p, F8Out{(bf16_t*)out, nullptr, nullptr, nullptr, N}, GatedAct{}, height, stream);
}

// codes [rows, 128 f8_blocks(I)] and scales [rows, f8_scale_stride(I)] of act(s g) (s u); w_rows: twice I up to a multiple of 32; score [rows] or null.
SHARPI_EXPORT int sharpi_fp8_tiles_gated(const void* x, const void* x_scales, int x_rows, const void* w_codes, const void* w_scales, int w_rows,
                                         void* codes, void* scales, int rows, int I, int K, const int* a_rows, const int* offsets, int groups, int along,
                                         const float* score, int act, float limit, int height, hipStream_t stream) {
  if (rows <= 0) return SHARPI_OK;
  const GatedAct ga{act, limit};
  if (I <= 0 || K <= 0 || w_rows != 2 * f8_padded_rows(I) || !act_known(ga) || ((uintptr_t)codes & 15)) return SHARPI_ERR_ARG;
  const F8Tiles p{(const uint8_t*)x, (const uint8_t*)x_scales, (const uint8_t*)w_codes, (const uint8_t*)w_scales, f8_blocks(K), w_rows, a_rows, offsets, rows, groups, along, 0, 0};
  if (!tiles_ok(p, x_rows)) return SHARPI_ERR_ARG;
  return launch_tiles<true>(p, F8Out{nullptr, (uint8_t*)codes, (uint8_t*)scales, score, I}, ga, height, stream);
}
