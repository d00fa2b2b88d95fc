// Products of few rows with weights in 8-bit floating point (fp8.h holds the format), weight-streaming: every block reads its tiles of the
// matrix once, with the streaming hint, and everything else is arranged around that.  Three forms:
//   plain   out[M, N] = q(x) W^T, bfloat16
//   gated   h = act(s g) (s u) with (g | u) = q(x) W^T, rounded to bfloat16: the first half of a feed-forward, for one matrix or for the
//           experts that a router picked (a block finds the rows of its expert among the picks itself)
//   sum     out[t] = sum_j w[t, j] q(h[t, j]) W_e^T over the token's picks e (and an always-on expert): the second half, with the sum
// q(.): a few rows of bfloat16 are quantised by every block that reads them, into LDS (no launch and no pass of their own; the weights' first loads are on
// their way meanwhile); other rows come as codes.
//
// Bound: bytes of the weights (13 rows of 202,048 x 5,120: 167 us, 6.3 TB/s; an expert of 8,192 x 5,120 and one always on, one token: 252 MB in 50 us with
// both launches).  Each wave takes blocks of 128 of k in turn, one 4 KB unit of a tile of 32 weight rows (or half of it)
// at a time through v_mfma_scale_f32_16x16x128: W is the A operand (rows = n), x the B operand (up to 16 rows a row block).  A lane ends
// up with four neighbouring n of one x row; the waves' sums meet in LDS and are added in wave order.
//
// The sum form deals all blocks of k of all experts that occur to S blocks a tile in equal shares, whatever the picks: a column tile has few
// blocks (160 of 32 columns at 5,120), the experts many bytes.  A column of the product is a token, whose row of h is looked up for each
// expert, so that all experts add up in the same accumulators.  Their partial sums go through memory; the last block of a tile to
// finish adds them in the order of the shares: the result does not depend on which that is.
#include "fp8.h"

namespace {

constexpr int FW = 8;                  // waves a block
constexpr int kFewRows = 64;           // rows (tokens) of a call at most: four row blocks
constexpr int kFewPairs = 512;         // (token, pick) pairs of a call at most
constexpr int kFewExperts = 1024;
constexpr int kStagedRows = 2;         // rows of bfloat16 that the kernels quantise themselves
constexpr int kLayerTiles = 2;         // half tiles a block of a layer's two products
constexpr int kRound = 2;              // (tile, row block) pairs that meet in LDS at a time

struct F8Matrix {
  const uint8_t* codes;    // [matrices][rows / 32][U][4096]
  const uint8_t* scales;   // [matrices][rows / 32][U4][32][4]
  int rows, U;             // rows of one matrix (a multiple of 32), blocks of 128 of k
};

// the picks of a call (ids null: one matrix, row = token)
struct F8Picks {
  const int* ids;          // [T, k]
  const float* w;          // [T, k] or null
  int T, k, E;
  int shared;              // one more matrix (number E) that every token goes through: rows T k + t
};

// A wave's view of one 16-row half tile of a matrix: addresses that the wave shares, and a lane's 32-bit offsets from them.
struct F8Lane {
  const uint8_t* codes;
  const uint8_t* scales;
  __device__ __forceinline__ void at(const F8Matrix& w, size_t matrix, int half_tile) {
    const int last = w.rows / 16 - 1, t = half_tile < last ? half_tile : last;      // (beyond the last: read, never stored)
    const size_t tile = matrix * (w.rows / 32) + (t >> 1);
    codes = w.codes + tile * w.U * kF8TileBytes + (t & 1) * 256;
    scales = w.scales + tile * ((w.U + 3) >> 2) * 128 + (t & 1) * 64;
  }
  // a lane's codes of row r, and the scale byte of row scale_row
  __device__ __forceinline__ i32x8 load(int u, int r, int g, int scale_row, int& s) const {
    const uint8_t* from = codes + (size_t)u * kF8TileBytes + (uint32_t)((g >> 1) * 2048 + (g & 1) * 512 + r * 16);
    const i32x4 a = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(from));
    const i32x4 b = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(from + 1024));
    s = (scales + (u >> 2) * 128 + (u & 3))[(uint32_t)scale_row * 4];
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
};

// Rows' blocks of 128 as codes in LDS, in the order of the operands: block b of n rows at [b][piece][group][row][16 bytes], its bytes behind one another.
struct F8Staged {
  uint8_t* codes;
  uint8_t* bytes;
  int n;                   // rows
  __device__ __forceinline__ i32x8 read(int b, int row, int g, int& s) const {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(codes + (((b * 2) * 4 + g) * n + row) * 16);
    const i32x4 hi = *reinterpret_cast<const i32x4*>(codes + (((b * 2 + 1) * 4 + g) * n + row) * 16);
    s = bytes[b * n + row];
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
};
// Quantises `tasks` blocks of rows of bfloat16 [.., K] into LDS, 16 lanes a block, four blocks of a lane group on their way at a time.  where(task, row, u, b, m): the
// row of x and its block u of a task, and where it is staged (block b, row m); row < 0: nothing is read.
template <typename F> __device__ __forceinline__ void stage_rows(const bf16_t* __restrict__ x, int K, int tasks, F8Staged to, const F& where) {
  const int l = threadIdx.x & 15;
  constexpr int kGroups = FW * kWave / 16, kFlight = 4;
  for (int t0 = threadIdx.x >> 4; t0 < tasks; t0 += kGroups * kFlight) {
    uint4 raw[kFlight];
    int b[kFlight], m[kFlight], row[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int t = t0 + i * kGroups;
      int u = 0;
      row[i] = -1;
      if (t < tasks) where(t, row[i], u, b[i], m[i]);
      const int k = u * kF8Block + l * 8;
      raw[i] = row[i] >= 0 && k < K ? *reinterpret_cast<const uint4*>(x + (size_t)row[i] * K + k) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      if (row[i] < 0) continue;                  // (16 lanes at once)
      const uint32_t d[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      uint32_t top = 0, bad = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = d[j] & 0x7fffu, hi = d[j] >> 16 & 0x7fffu;
        top = lo < 0x7f80u && lo > top ? lo : top;
        top = hi < 0x7f80u && hi > top ? hi : top;
        bad |= (lo >= 0x7f80u ? 1u : 0u) << (2 * j) | (hi >= 0x7f80u ? 1u : 0u) << (2 * j + 1);
      }
      float t = __uint_as_float(top << 16);
      t = fmaxf(t, row_rotated<8>(t));
      t = fmaxf(t, row_rotated<4>(t));
      t = fmaxf(t, row_rotated<2>(t));
      t = fmaxf(t, row_rotated<1>(t));
      const int s = f8_scale_of(__float_as_uint(t));
      const float scale = f8_scale_value(s);
      uint32_t c[2] = {f8_codes4(d[0], d[1], scale), f8_codes4(d[2], d[3], scale)};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (bad >> j & 1) c[j / 4] = (c[j / 4] & ~(0xffu << (j % 4 * 8))) | kF8Nan << (j % 4 * 8);
      *reinterpret_cast<uint2*>(to.codes + (((b[i] * 2 + (l >> 1 & 1)) * 4 + (l >> 2)) * to.n + m[i]) * 16 + (l & 1) * 8) = make_uint2(c[0], c[1]);
      if (l == 0) to.bytes[b[i] * to.n + m[i]] = (uint8_t)s;
    }
  }
}

// A lane's 32 codes of a row's block u of k, from memory.
struct F8Row {
  i32x4 a, b;
  int byte;
  // OFFSET: of the row's lane piece and of its bytes, 32 bits where the rows lie within 4 GB
  template <typename OFFSET> __device__ __forceinline__ void load(const void* x, const uint8_t* scales, OFFSET at, OFFSET scale_at, int u) {
    const uint8_t* p = (const uint8_t*)x + (size_t)u * kF8Block + at;
    a = *reinterpret_cast<const i32x4*>(p);
    b = *reinterpret_cast<const i32x4*>(p + 16);
    byte = (scales + u)[scale_at];
  }
  __device__ __forceinline__ i32x8 codes(int& s) const {
    s = byte;
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
};

__device__ __forceinline__ f32x4 f8_product(const i32x8& w, const i32x8& x, const f32x4& c, int ws, int xs) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, 0, ws, 0, xs);
}

// The same with every product and sum in float: codes widened to bfloat16, which holds them, and both scales on the block's sum, whose exponent holds
// them together (a weight's scale times its code may lie beyond bfloat16, and beyond float its product with a row's code).  For results that are
// quantised again: what the scaled instruction leaves out moves 1 value in 390 across a border of e4m3 (float sums 1 in 170,000 and fewer), and the
// layer's error against 64 bits was 1.5 times that of the same sums in float.  The widening is hidden by the weights' way from memory.
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
__device__ __forceinline__ bf16x8 f8_wide(int lo, int hi) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, 1.0f, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// ws: of the four rows whose sums a lane ends up with, g * 4 + 0 .. 3, the four neighbouring lanes hold a scale byte each.
template <int I> __device__ __forceinline__ int f8_byte_of(int ws) { return __builtin_amdgcn_update_dpp(0, ws, I * 0x55, 0xf, 0xf, true); }
template <int R> __device__ __forceinline__ void f8_product_in_float(const i32x8 (&w)[R], const int (&ws)[R], const i32x8& x, int xs, f32x4* acc, int step) {
  f32x4 sum[R];
#pragma unroll
  for (int t = 0; t < R; ++t) sum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bf16x8 xw = f8_wide(x[2 * j], x[2 * j + 1]);
#pragma unroll
    for (int t = 0; t < R; ++t) sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f8_wide(w[t][2 * j], w[t][2 * j + 1]), xw, sum[t], 0, 0, 0);
  }
#pragma unroll
  for (int t = 0; t < R; ++t) {
    const int b[4] = {f8_byte_of<0>(ws[t]), f8_byte_of<1>(ws[t]), f8_byte_of<2>(ws[t]), f8_byte_of<3>(ws[t])};
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t * step][i] += f8_scaled(sum[t][i], b[i] + xs);
  }
}

// Four neighbouring columns from n on of one row of `columns`.
__device__ __forceinline__ void store_columns(bf16_t* row, int n, int columns, const f32x4& v) {
  if (n + 4 <= columns && ((uintptr_t)(row + n) & 7) == 0) {
    *reinterpret_cast<uint2*>(row + n) = make_uint2(f32_to_bf16_pair(v[0], v[1]), f32_to_bf16_pair(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < columns) row[n + i] = f32_to_bf16(v[i]);
  }
}

// plain and gated.  R half tiles a block: of distinct columns (plain), or R / 2 of gate columns and the up columns beside them (gated).
// n_out: columns of the result that exist; stride: of a stored row (gated: the columns from n_out to it are zeros, as their weights are).
// STAGED: x is bfloat16, up to kStagedRows rows, quantised into LDS, `turn` of an expert's at a time; else codes.
template <int R, int MB, bool STAGED, bool GATED>
__global__ __launch_bounds__(FW* kWave, MB > 1 ? 2 : 4) void fp8_few_kernel(const void* __restrict__ x, const uint8_t* __restrict__ x_scales, F8Matrix W,
                                                                            bf16_t* __restrict__ out, int n_out, int stride, int M, int K, GatedAct act,
                                                                            F8Picks pk, int* __restrict__ clear, int n_clear, int turn) {
  static_assert(!STAGED || MB == 1, "staged rows are one row block");
  extern __shared__ __attribute__((aligned(16))) uint8_t staged_bytes[];
  constexpr int TG = GATED ? R / 2 : R;
  constexpr int RT = GATED ? R : kRound;
  __shared__ f32x4 red[FW][RT][kWave];
  __shared__ short members[GATED ? kFewPairs + kFewRows : 1];
  __shared__ int flags[GATED ? kFewExperts : 1];
  __shared__ int n_members;
  const int lane = threadIdx.x & (kWave - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  int rows = M, expert = 0;
  const bool picked = GATED && pk.ids != nullptr;
  if constexpr (GATED) {
    if (clear && blockIdx.x == 0 && blockIdx.y == 0)          // the counters of the sum behind this launch
      for (int i = threadIdx.x; i < n_clear; i += FW * kWave) clear[i] = 0;
  }
  if (picked) {
    // Group 0 is the always-on matrix, if there is one; the others are experts, all of them where there are as many groups, else the
    // distinct ones among the picks in their order (the groups that find none are the grid's last blocks).
    const int n_pairs = pk.T * pk.k, group = (int)blockIdx.y - pk.shared;
    if (group < 0) {
      expert = pk.E;
      rows = pk.T;
    } else {
      if ((int)gridDim.y - pk.shared == pk.E) {
        expert = group;
      } else {
        int mine[kFewPairs / (FW * kWave)];
#pragma unroll
        for (int i = 0; i < kFewPairs / (FW * kWave); ++i) {
          const int p = i * FW * kWave + threadIdx.x;
          mine[i] = p < n_pairs ? pk.ids[p] : -1;
        }
        for (int i = threadIdx.x; i < pk.E; i += FW * kWave) flags[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kFewPairs / (FW * kWave); ++i)
          if ((unsigned)mine[i] < (unsigned)pk.E) flags[mine[i]] = 1;
        __syncthreads();
        int before = 0;
        expert = -1;
        for (int c = 0; c < pk.E && expert < 0; c += kWave) {
          unsigned long long m = __builtin_amdgcn_ballot_w64(c + lane < pk.E && flags[c + lane] != 0);
          const int n = __popcll(m);
          if (group < before + n) {
            for (int i = before; i < group; ++i) m &= m - 1;
            expert = c + __ffsll((long long)m) - 1;
          }
          before += n;
        }
      }
      expert = __builtin_amdgcn_readfirstlane(expert);
      if (expert < 0) return;                   // (the same for the block)
      if (w == 0) {
        int n = 0;
        for (int c = 0; c < n_pairs; c += kWave) {
          const bool mine = c + lane < n_pairs && pk.ids[c + lane] == expert;
          const unsigned long long m = __builtin_amdgcn_ballot_w64(mine);
          if (mine) members[n + __popcll(m & ((1ull << lane) - 1ull))] = (short)(c + lane);
          n += __popcll(m);
        }
        if (lane == 0) n_members = n;
      }
      __syncthreads();
      rows = __builtin_amdgcn_readfirstlane(n_members);
    }
  }
  if (rows <= 0) return;
  const bool routed = picked && expert < pk.E;
  auto out_row = [&](int m) { return routed ? (int)members[m] : picked ? pk.T * pk.k + m : m; };
  auto x_row = [&](int m) { return routed ? members[m] / pk.k : m; };
  const int group_rows = STAGED ? turn : 16 * MB;
  for (int rb = 0; rb < rows; rb += group_rows) {
    const int here = min(rows - rb, group_rows);            // rows of this turn
    const F8Staged st{staged_bytes, staged_bytes + W.U * kF8Block * here, here};
    // (staged: the row; codes: offsets, of up to 64 rows)
    uint32_t xr[MB], xsr[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const uint32_t row = STAGED ? min(r, here - 1) : x_row(rb + min(mb * 16 + r, here - 1));
      xr[mb] = STAGED ? row : row * (W.U * kF8Block) + g * 32;
      xsr[mb] = row * f8_scale_stride(K);
    }
    const int n_base = blockIdx.x * 16 * TG;
    F8Lane wl[R];
    // (of a gated matrix the up rows begin at half its rows, a multiple of 32: half tile rows / 32)
#pragma unroll
    for (int t = 0; t < R; ++t)
      wl[t].at(W, expert, n_base / 16 + t % TG + (GATED && t >= TG ? W.rows / 32 : 0));
    f32x4 acc[R][MB];
#pragma unroll
    for (int t = 0; t < R; ++t)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) acc[t][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Unit {
      i32x8 wf[R];
      int ws[R];
      F8Row xf[STAGED ? 1 : MB];
    };
    auto load_unit = [&](int u, Unit& un) {
#pragma unroll
      for (int t = 0; t < R; ++t) un.wf[t] = wl[t].load(u, r, g, GATED ? g * 4 + (r & 3) : r, un.ws[t]);
      if constexpr (!STAGED) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) un.xf[mb].load(x, x_scales, xr[mb], xsr[mb], u);     // (a row block without rows reads the last row)
      }
    };
    auto use_unit = [&](int u, Unit& un) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        int xs;
        const i32x8 c = STAGED ? st.read(u, (int)xr[0], g, xs) : un.xf[STAGED ? 0 : mb].codes(xs);
        if constexpr (GATED) {
          f8_product_in_float<R>(un.wf, un.ws, c, xs, &acc[0][mb], MB);
        } else {
#pragma unroll
          for (int t = 0; t < R; ++t) acc[t][mb] = f8_product(un.wf[t], c, acc[t][mb], un.ws[t], xs);
        }
      }
    };
    Unit a, b;
    int u = w;
    if (u < W.U) load_unit(u, a);
    if constexpr (STAGED) {
      if (rb > 0) __syncthreads();                          // (the turn before has been read)
      stage_rows((const bf16_t*)x, K, here * W.U, st, [&](int task, int& row, int& block, int& to, int& m) {
        m = task / W.U;
        block = to = task - m * W.U;
        row = x_row(rb + m);
      });
      __syncthreads();
    }
    for (; u + 2 * FW < W.U; u += 2 * FW) {
      load_unit(u + FW, b);
      use_unit(u, a);
      load_unit(u + 2 * FW, a);
      use_unit(u + FW, b);
    }
    if (u + FW < W.U) {
      load_unit(u + FW, b);
      use_unit(u, a);
      use_unit(u + FW, b);
    } else if (u < W.U) {
      use_unit(u, a);
    }

    if constexpr (GATED) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        if (mb > 0 && mb * 16 >= here) continue;
        __syncthreads();
#pragma unroll
        for (int t = 0; t < R; ++t) red[w][t][lane] = acc[t][mb];
        __syncthreads();
        if (w < TG) {
          f32x4 gv = red[0][w][lane], uv = red[0][w + TG][lane];
#pragma unroll
          for (int ww = 1; ww < FW; ++ww) {
            gv += red[ww][w][lane];
            uv += red[ww][w + TG][lane];
          }
          const int m = mb * 16 + r, n = n_base + w * 16 + g * 4;
          if (m < here && n < stride) {
            const int orow = out_row(rb + m);
            const bool scaled = routed && pk.w != nullptr;
            const float sc = scaled ? pk.w[orow] : 1.0f;
            f32x4 o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = f8_unit(act, gv[i] * sc, uv[i] * sc);
            store_columns(out + (size_t)orow * stride, n, stride, o);
          }
        }
      }
    } else {
#pragma unroll
      for (int p0 = 0; p0 < R * MB; p0 += kRound) {
        bool any = false;
#pragma unroll
        for (int p = 0; p < kRound; ++p) any = any || (p0 + p < R * MB && (p0 + p) % MB * 16 < here);
        if (!any) continue;
        __syncthreads();
#pragma unroll
        for (int p = 0; p < kRound; ++p)
          if (p0 + p < R * MB) red[w][p][lane] = acc[(p0 + p) / MB][(p0 + p) % MB];
        __syncthreads();
        if (w < kRound && p0 + w < R * MB) {
          const int t = (p0 + w) / MB, mb = (p0 + w) % MB;
          f32x4 v = red[0][w][lane];
#pragma unroll
          for (int ww = 1; ww < FW; ++ww) v += red[ww][w][lane];
          const int m = mb * 16 + r, n = n_base + t * 16 + g * 4;
          if (m < here && n < n_out) store_columns(out + (size_t)(rb + m) * stride, n, n_out, v);
        }
      }
    }
  }
}

// The sum over a token's picks.  R half tiles of columns a block, MB row blocks of tokens; blockIdx.y: the share of the blocks of k.
// part [S][tiles][MB][R][64 lanes] float4, counters [tiles] zero before the launch (both unused if S is 1).
// STAGED: h is bfloat16, up to kStagedRows tokens, quantised into LDS `chunk` blocks of k (a multiple of 2 FW) at a time; else codes.
template <int R, int MB, bool STAGED>
__global__ __launch_bounds__(FW* kWave, MB > 1 ? 2 : 4) void fp8_sum_kernel(const void* __restrict__ h, const uint8_t* __restrict__ h_scales, F8Matrix W,
                                                                            bf16_t* __restrict__ out, int n_out, int K, F8Picks pk, int weighted,
                                                                            f32x4* __restrict__ part, int* __restrict__ counters, int chunk) {
  static_assert(!STAGED || MB == 1, "staged rows are one row block");
  extern __shared__ __attribute__((aligned(16))) uint8_t staged_bytes[];
  __shared__ f32x4 red[FW][kRound][kWave];
  __shared__ short ids[kFewPairs];              // (-1: a pick of no expert)
  __shared__ float wts[kFewPairs];
  __shared__ int occurs[kFewExperts];           // times that one token picks the expert, at most
  __shared__ int entry[kFewPairs + 1];          // expert | occurrence << 16
  __shared__ int n_entries, is_last;
  const int lane = threadIdx.x & (kWave - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n_pairs = pk.ids ? pk.T * pk.k : 0;
  if (pk.ids) {
    for (int i = threadIdx.x; i < n_pairs; i += FW * kWave) {
      const int e = pk.ids[i];
      ids[i] = (unsigned)e < (unsigned)pk.E ? (short)e : (short)-1;
      if (weighted) wts[i] = pk.w[i];
    }
    for (int i = threadIdx.x; i < pk.E; i += FW * kWave) occurs[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n_pairs; i += FW * kWave) {
      const int e = ids[i];
      int n = 1;
      for (int j = i / pk.k * pk.k; j < i; ++j) n += ids[j] == e;
      if (e >= 0) atomicMax(&occurs[e], n);
    }
    __syncthreads();
    if (w == 0) {                               // (expert, occurrence) entries in the experts' order, the always-on one last
      int n = 0;
      for (int c = 0; c < pk.E; c += kWave) {
        const int mine = c + lane < pk.E ? occurs[c + lane] : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
          const int up = __shfl_up(upto, o, kWave);
          if (lane >= o) upto += up;
        }
        for (int i = 0; i < mine; ++i) entry[n + upto - mine + i] = (c + lane) | i << 16;
        n += __shfl(upto, kWave - 1, kWave);
      }
      if (pk.shared && lane == 0) entry[n] = pk.E;
      if (lane == 0) n_entries = n + pk.shared;
    }
    __syncthreads();
  }
  const int entries = pk.ids ? __builtin_amdgcn_readfirstlane(n_entries) : 1;
  const int S = gridDim.y, share = blockIdx.y, all = entries * W.U;      // (entries x blocks of k: up to 513 x 2^17)
  const int first = (int)((long long)all * share / S), end = (int)((long long)all * (share + 1) / S);
  const int n_base = blockIdx.x * 16 * R;

  f32x4 total[R][MB];
#pragma unroll
  for (int t = 0; t < R; ++t)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) total[t][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
  // the row of h that a token has for an entry (-1: none) and its weight
  auto row_of = [&](int code, int tok, float& weight) {
    weight = 1.f;
    if (tok >= pk.T) return -1;
    if (!pk.ids) return tok;
    const int e = code & 0xffff, occurrence = code >> 16;
    if (e == pk.E) return n_pairs + tok;
    int row = -1, seen = 0;
    for (int j = 0; j < pk.k; ++j) {
      const int p = tok * pk.k + j;
      if (ids[p] == e) {
        if (seen == occurrence) {
          row = p;
          if (weighted) weight = wts[p];
        }
        ++seen;
      }
    }
    return row;
  };
  auto code_of = [&](int at) { return pk.ids ? entry[at] : 0; };
  struct Unit {
    i32x8 wf[R];
    int ws[R];
    F8Row xf[STAGED ? 1 : MB];
    float weight[MB];
    int row[MB];
  };
  auto load_unit = [&](int i, Unit& un) {
    i = min(i, end - 1);                            // (past the share: its last block once more, for nobody)
    const int at = i / W.U, u = i - at * W.U, code = __builtin_amdgcn_readfirstlane(code_of(at));
#pragma unroll
    for (int t = 0; t < R; ++t) {
      F8Lane wl;
      wl.at(W, code & 0xffff, n_base / 16 + t);
      un.wf[t] = wl.load(u, r, g, r, un.ws[t]);
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      un.row[mb] = row_of(code, mb * 16 + r, un.weight[mb]);
      const size_t row = max(un.row[mb], 0);
      if constexpr (!STAGED) un.xf[mb].load(h, h_scales, row * (W.U * kF8Block) + g * 32, row * f8_scale_stride(K), u);      // (row 0: read for a token without this expert, never added)
    }
  };
  const F8Staged st{staged_bytes, staged_bytes + chunk * kF8Block * pk.T, pk.T};
  auto use_unit = [&](int staged_block, Unit& un) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      int xs;
      const i32x8 c = STAGED ? st.read(staged_block, min(r, pk.T - 1), g, xs) : un.xf[STAGED ? 0 : mb].codes(xs);
#pragma unroll
      for (int t = 0; t < R; ++t) {
        const f32x4 v = f8_product(un.wf[t], c, f32x4{0.f, 0.f, 0.f, 0.f}, un.ws[t], xs);
#pragma unroll
        for (int i = 0; i < 4; ++i) total[t][mb][i] = un.row[mb] >= 0 ? fmaf(un.weight[mb], v[i], total[t][mb][i]) : total[t][mb][i];
      }
    }
  };
  if (first < end) {
    Unit a, b;
    load_unit(first + w, a);
    for (int c0 = first; c0 < end; c0 += chunk) {
      if constexpr (STAGED) {
        if (c0 > first) __syncthreads();            // (the chunk before has been read)
        const int blocks = min(chunk, end - c0);
        stage_rows((const bf16_t*)h, K, blocks * pk.T, st, [&](int task, int& row, int& block, int& to, int& m) {
          to = task / pk.T;
          m = task - to * pk.T;
          const int at = (c0 + to) / W.U;
          float weight;
          block = c0 + to - at * W.U;
          row = row_of(code_of(at), m, weight);
        });
        __syncthreads();
      }
      for (int j = w; j < chunk; j += 2 * FW) {
        const int i = c0 + j;
        if (i >= end) break;
        load_unit(i + FW, b);
        use_unit(j, a);
        if (i + FW >= end) break;
        load_unit(i + 2 * FW, a);
        use_unit(j + FW, b);
      }
    }
  }

  auto store = [&](int t, int mb, const f32x4& v) {
    const int tok = mb * 16 + r, n = n_base + t * 16 + g * 4;
    if (tok < pk.T && n < n_out) store_columns(out + (size_t)tok * n_out, n, n_out, v);
  };
  // part: [share][tile][pair p][lane]
  const size_t tile_parts = (size_t)R * MB * kWave, share_parts = (size_t)gridDim.x * tile_parts;
#pragma unroll
  for (int p0 = 0; p0 < R * MB; p0 += kRound) {
    __syncthreads();
#pragma unroll
    for (int p = 0; p < kRound; ++p)
      if (p0 + p < R * MB) red[w][p][lane] = total[(p0 + p) / MB][(p0 + p) % MB];
    __syncthreads();
    if (w < kRound && p0 + w < R * MB) {
      f32x4 v = red[0][w][lane];
#pragma unroll
      for (int ww = 1; ww < FW; ++ww) v += red[ww][w][lane];
      if (S == 1) store((p0 + w) / MB, (p0 + w) % MB, v);
      else {
        float* dst = reinterpret_cast<float*>(part + share * share_parts + blockIdx.x * tile_parts + (size_t)(p0 + w) * kWave + lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) __hip_atomic_store(dst + i, v[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (S == 1) return;
  // What the block wrote is in memory before its ticket counts; who draws the last ticket adds the shares up in their order.  The shares are written and
  // read as words that all dies see (agent scope), so a wait for the wave's own stores is all that the ticket needs: a fence writes back the
  // whole L2 of the die, every wave anew (84 MB of weights in 480 blocks: 160 us).
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) is_last = __hip_atomic_fetch_add(&counters[blockIdx.x], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == S - 1;
  __syncthreads();
  if (!is_last) return;
  for (int p = w; p < R * MB; p += FW) {
    const float* src = reinterpret_cast<const float*>(part + blockIdx.x * tile_parts + (size_t)p * kWave + lane);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += __hip_atomic_load(src + s * share_parts * 4 + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    store(p / MB, p % MB, v);
  }
}

// x operand of a call: codes, or (up to kStagedRows rows) bfloat16 whose runs of eight lie at 16-byte addresses
enum : int { X_BF16 = DT_BF16, X_CODES = 2 };
constexpr int kStagedMost = 48 * 1024;          // bytes of LDS for staged rows
constexpr int kMostAcross = 0x7fffff;           // blocks of a launch along x (of 512 threads each, of which there are at most 2^32)
bool rows_ok(const void* x, int kind, int M, int K) {
  if (((uintptr_t)x & 15) != 0) return false;
  return kind == X_CODES || (kind == X_BF16 && K % 8 == 0 && M <= kStagedRows);
}
int staged_size(int rows, int blocks) { return rows * blocks * (kF8Block + 1) + 16; }
bool matrix_ok(const F8Matrix& W, long long matrices) {
  return W.rows > 0 && W.rows % kF8Tile == 0 && W.U > 0 && matrices > 0 && (long long)W.rows * W.U < 0x7fffffffLL && !(((uintptr_t)W.codes) & 15);
}

}  // namespace

// out [M, N] bfloat16 = q(x [M, K]) W^T, M <= 64.  kind: X_*; w_rows: stored rows of W (N up to a multiple of 32); R 1 or 2 half tiles a block.
SHARPI_EXPORT int sharpi_fp8_few(const void* x, const void* x_scales, int kind, const void* w_codes, const void* w_scales, int w_rows, void* out,
                                 int M, int N, int K, int R, hipStream_t stream) {
  if (M <= 0) return SHARPI_OK;
  const F8Matrix W{(const uint8_t*)w_codes, (const uint8_t*)w_scales, w_rows, f8_blocks(K)};
  if ((R != 1 && R != 2) || M > kFewRows || N <= 0 || K <= 0 || K >= kF8MostK || w_rows != f8_padded_rows(N) || !matrix_ok(W, 1) || !rows_ok(x, kind, M, K)) return SHARPI_ERR_ARG;
  const int mb = M <= 16 ? 1 : M <= 32 ? 2 : 4, groups = ceil_div(N, 16 * R);
  const int lds = kind == X_CODES ? 0 : staged_size(M, W.U);
  if (lds > kStagedMost || groups > kMostAcross) return SHARPI_ERR_ARG;
  const dim3 grid((unsigned)groups), block(FW * kWave);
#define FF(RV, MBV, STG) \
  fp8_few_kernel<RV, MBV, STG, false><<<grid, block, lds, stream>>>(x, (const uint8_t*)x_scales, W, (bf16_t*)out, N, N, M, K, GatedAct{}, F8Picks{}, nullptr, 0, M)
#define FF_X(RV)                          \
  if (kind != X_CODES) FF(RV, 1, true);   \
  else if (mb == 1) FF(RV, 1, false);     \
  else if (mb == 2) FF(RV, 2, false);     \
  else FF(RV, 4, false)
  if (R == 1) { FF_X(1); }
  else { FF_X(2); }
#undef FF_X
#undef FF
  SHARPI_CHECK_LAUNCH();
  return SHARPI_OK;
}

static bool picks_ok(const F8Picks& p) {
  if (p.T <= 0 || p.T > kFewRows || p.E <= 0 || p.E > kFewExperts) return false;
  if (!p.ids) return p.E == 1 && !p.shared;
  return p.k > 0 && (long long)p.T * p.k <= kFewPairs;
}

// h [T k (+ T), stride] bfloat16 = act(s g) (s u) of the picked experts, pair by pair, then (shared) a row per token through matrix E; ids null: one
// matrix, h [T, stride].  I: columns that exist; stride: I up to a multiple of 8; w_rows: twice I up to a multiple of 32.  wts: the pairs' s, or null.
// clear [n_clear]: set to zero (the counters of the launch behind).
SHARPI_EXPORT int sharpi_fp8_few_gated(const void* x, const void* x_scales, int kind, const void* w_codes, const void* w_scales, int w_rows, void* h,
                                       int stride, const int* ids, const float* wts, int T, int k, int E, int shared, int I, int K, int act, float limit,
                                       int* clear, int n_clear, hipStream_t stream) {
  if (T <= 0) return SHARPI_OK;
  const F8Matrix W{(const uint8_t*)w_codes, (const uint8_t*)w_scales, w_rows, f8_blocks(K)};
  const F8Picks pk{ids, wts, T, k, E, shared ? 1 : 0};
  const GatedAct ga{act, limit};
  if (I <= 0 || K <= 0 || K >= kF8MostK || w_rows != 2 * f8_padded_rows(I) || stride != (I + 7) / 8 * 8 || !act_known(ga) || !picks_ok(pk) ||
      !matrix_ok(W, E + pk.shared) || !rows_ok(x, kind, T, K) || ((uintptr_t)h & 15)) return SHARPI_ERR_ARG;
  const int mb = T <= 16 ? 1 : T <= 32 ? 2 : 4;
  const int groups = ids ? (T * k < E ? T * k : E) + pk.shared : 1, column_groups = ceil_div(I, 8 * kLayerTiles);
  const int lds = kind == X_CODES ? 0 : staged_size(T, W.U);       // (rows of a turn: the tokens')
  if (lds > kStagedMost || column_groups > kMostAcross) return SHARPI_ERR_ARG;
  const dim3 grid((unsigned)column_groups, (unsigned)groups), block(FW * kWave);
#define FG(MBV, STG) \
  fp8_few_kernel<kLayerTiles, MBV, STG, true><<<grid, block, lds, stream>>>(x, (const uint8_t*)x_scales, W, (bf16_t*)h, I, stride, T, K, ga, pk, clear, n_clear, T)
  if (kind != X_CODES) FG(1, true);
  else if (mb == 1) FG(1, false);
  else if (mb == 2) FG(2, false);
  else FG(4, false);
#undef FG
  SHARPI_CHECK_LAUNCH();
  return SHARPI_OK;
}

// out [T, N] bfloat16 = the sum over the picks of q(h row) W_e^T (times the pair's weight if wts is given), plus the always-on expert's.
// h [T k (+ T), K]: bfloat16 (up to kStagedRows tokens, K a multiple of 8) or codes.  S shares of the blocks of k for each tile of 16 kLayerTiles columns; part: S x
// tiles x 1 KB x kLayerTiles x row blocks; counters [tiles] zero.
SHARPI_EXPORT int sharpi_fp8_few_sum(const void* h, const void* h_scales, int kind, const void* w_codes, const void* w_scales, int w_rows, void* out, const int* ids, const float* wts,
                                     int T, int k, int E, int shared, int N, int K, int S, void* part, int* counters, hipStream_t stream) {
  if (T <= 0) return SHARPI_OK;
  const F8Matrix W{(const uint8_t*)w_codes, (const uint8_t*)w_scales, w_rows, f8_blocks(K)};
  const F8Picks pk{ids, wts, T, k, E, shared ? 1 : 0};
  if (N <= 0 || K <= 0 || K >= kF8MostK || w_rows != f8_padded_rows(N) || !picks_ok(pk) || !matrix_ok(W, E + pk.shared) || !rows_ok(h, kind, T, K) || S < 1 ||
      S > 0xffff || (S > 1 && (!part || !counters)) || ceil_div(N, 16 * kLayerTiles) > kMostAcross) return SHARPI_ERR_ARG;
  const int mb = T <= 16 ? 1 : T <= 32 ? 2 : 4;
  const dim3 grid((unsigned)ceil_div(N, 16 * kLayerTiles), (unsigned)S), block(FW * kWave);
  constexpr int chunk = 4 * FW;                       // blocks of k staged at a time: up to 16 KB of rows
  const int lds = kind == X_CODES ? 0 : staged_size(T, chunk);
#define FS(MBV, STG) \
  fp8_sum_kernel<kLayerTiles, MBV, STG><<<grid, block, lds, stream>>>(h, (const uint8_t*)h_scales, W, (bf16_t*)out, N, K, pk, wts != nullptr, (f32x4*)part, counters, \
                                                             STG ? chunk : 0x40000000)
  if (kind != X_CODES) FS(1, true);
  else if (mb == 1) FS(1, false);
  else if (mb == 2) FS(2, false);
  else FS(4, false);
#undef FS
  SHARPI_CHECK_LAUNCH();
  return SHARPI_OK;
}
