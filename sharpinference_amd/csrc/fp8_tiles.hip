// Products of many rows with weights in 8-bit floating point (fp8.h holds the format), in tiles on the scaled matrix instruction: one matrix, or
// the experts of a routing's sorted row list.  Two forms:
//   plain   out[row, :] = rows[row] W_e^T, bfloat16
//   gated   act(s g) (s u) with (g | u) the product, rounded to bfloat16 and quantised again: codes and scale bytes of the rows that the
//           second half of a feed-forward reads.  A block's 128 output columns are one block of the format, so the epilogue has what
//           it needs, and neither (g | u) nor the unquantised rows go to memory.
// Every output is one chain over k in ascending order: a row's result does not depend on which rows share its tile.
#include <type_traits>

#include "fp8.h"
#include "lds_loads.h"

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
  uint32_t x_bytes;          // of x's codes (with a_rows)
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

// Where 16-byte piece `piece` of row `row` of a stage is kept: the pieces of a wave's read fall into different 16-byte groups of the banks.
__device__ __forceinline__ int row_piece(int row, int piece) { return piece ^ ((row >> 1) & 7); }

// MT: groups of 32 rows a wave; a tile has 64 MT rows.
template <int MT, bool GATED>
__global__ __launch_bounds__(TW* kWave, 2) void fp8_tiles_kernel(F8Tiles p, F8Out o, GatedAct act) {
  constexpr int TM = 64 * MT;
  // The rings: of tall tiles two stages of rows (128 of k) and four steps of weights (64 of k), filled a step at a time, weights three steps ahead; of
  // tiles of up to 128 rows, whose steps are short beside a latency, three stages of both, filled a stage at a time.
  constexpr bool STAGED = MT <= 2;
  constexpr int RS = STAGED ? 3 : 2;
  constexpr int kWStep = 16384, kXStage = TM * kF8Block, kXAt = 2 * RS * kWStep, kSAt = kXAt + RS * kXStage;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kSAt + 3 * 2048];
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
  const int half = p.w_rows / 64;                // gated: tiles of the gate rows
  const bool exists = !GATED || nblock * (kTileCols / 64) + wc < half;
  // Loads into LDS.  Weights: wave wid brings tile wid of the block's eight (gated: a wave column's gate tile, then its up tile), a step of 64 of k
  // is 2 KB of it on end.  Rows: a load brings 8 rows of 128 bytes (a stage: two steps), lane l row l / 8 at place l % 8, their 16-byte pieces
  // exchanged by row bits (row_piece).  Rows behind the last read it again; what they give is never stored.  Scales: a chunk of four blocks of k
  // is a word a row; waves 0 to 3 bring those of 64 rows each, waves 4 to 7 those of two weight tiles each.
  auto block_tile = [&](int lt) {
    if constexpr (GATED) return min(nblock * (kTileCols / 64) + lt / 2, half - 1) + lt % 2 * half;
    else return min(nblock * (kTileCols / 32) + lt, p.w_rows / 32 - 1);
  };
  const size_t w_at = (size_t)e * (p.w_rows / 32);
  const u32x4 wb = buffer_of(p.w + (w_at + block_tile(wid)) * p.U * kF8TileBytes, (uint32_t)p.U * kF8TileBytes);
  const uint32_t lds0 = lds_address((const char*)smem);
  const uint32_t x_stride = (uint32_t)p.U * kF8Block;
  const size_t x_first = p.a_rows ? 0 : row0;             // (rows in a row: the tile's own piece of x, at any distance)
  const uint32_t x_bytes = p.a_rows ? p.x_bytes : (uint32_t)(row_end - row0) * x_stride;
  const u32x4 xb = buffer_of(p.x + x_first * x_stride, x_bytes);
  auto x_row = [&](int lrow) {
    const int row = min(row0 + lrow, row_end - 1);
    return !p.a_rows ? row - row0 : sorted ? p.a_rows[row] : row - p.rows;
  };
  constexpr int XL = MT;                                  // loads of rows a wave and stage
  const int steps = 2 * p.U;
  const uint32_t w_off[2] = {(uint32_t)lane * 16, (uint32_t)lane * 16 + 1024};
  auto load_w = [&](int s, int place) {
    const uint32_t at[2] = {lds0 + place * kWStep + wid * 2048, lds0 + place * kWStep + wid * 2048 + 1024};
    load_two_to_lds<false>(wb, w_off[0], w_off[1], min(s, steps - 1) * 2048, at[0], at[1]);
  };
#pragma unroll
  for (int s = 0; s < (STAGED ? 2 * RS - 2 : 3); ++s) load_w(s, s);      // (on their way while the rows' places are looked up)
  uint32_t x_off[XL], xs_off;
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int lrow = (wid * XL + i) * 8 + (lane >> 3);
    x_off[i] = (uint32_t)x_row(lrow) * x_stride + row_piece(lrow, lane & 7) * 16;
  }
  // scales: the wave's own buffer
  u32x4 sb;
  if (wid < 4) {
    const int lrow = min(wid, MT - 1) * 64 + lane;
    xs_off = (uint32_t)x_row(lrow) * (U4 * 4);
    sb = buffer_of(p.xs + x_first * (U4 * 4), p.a_rows ? (uint32_t)(p.x_bytes / x_stride) * (U4 * 4) : (uint32_t)(row_end - row0) * (U4 * 4));
  } else {
    const int lt = (wid - 4) * 2;
    const int t0 = block_tile(lt), t1 = block_tile(lt + 1);
    const uint8_t* base = p.ws + w_at * U4 * 128;
    const int low = min(t0, t1);                          // (the descriptor begins at the lower of the two tiles)
    xs_off = (uint32_t)((lane < 32 ? t0 : t1) - low) * (U4 * 128) + (lane & 31) * 4;
    sb = buffer_of(base + (size_t)low * U4 * 128, (uint32_t)(max(t0, t1) - low + 1) * (U4 * 128));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sb[i] = (uint32_t)__builtin_amdgcn_readfirstlane(sb[i]);
  const uint32_t s_lds = lds0 + kSAt + (wid < 4 ? min(wid, MT - 1) * 256 : 1024 + (wid - 4) * 256);
  const uint32_t s_step = wid < 4 ? 4 : 128;
  // waited for here: the compiler's own waits must not fall among the loads below, which it does not know of
#pragma unroll
  for (int i = 0; i < XL; ++i) asm volatile("" : "+v"(x_off[i]));
  asm volatile("" : "+v"(xs_off));
  // the scales of the chunk behind chunk c, once a chunk; the other blocks' loads go where nobody reads
  auto load_s = [&](int c, bool first) { load_words_to_lds(sb, xs_off, min(c + 1, U4 - 1) * s_step, s_lds + (first ? ((c + 1) & 1) * 2048 : 4096)); };
  auto load_x = [&](int c, int place) {
    uint32_t at[XL];
#pragma unroll
    for (int i = 0; i < XL; ++i) at[i] = lds0 + kXAt + place * kXStage + (wid * XL + i) * 1024;
    bring_all_to_lds<true, XL>(xb, x_off, min(c, p.U - 1) * kF8Block, at);
  };
  load_s(-1, true);
#pragma unroll
  for (int c = 0; c < RS - 1; ++c) load_x(c, c);

  f32x16 acc[2][MT];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][m][i] = 0.f;
  // operand addresses: piece q of a lane's 32 bytes of half hh
  int w_lds[2], x_lds[2][2];
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    w_lds[hh] = wc * 4096 + lane * 16 + hh * kWStep;
#pragma unroll
    for (int q = 0; q < 2; ++q) x_lds[hh][q] = kXAt + (wr * MT * 32 + r) * 128 + row_piece(r, hh * 4 + g * 2 + q) * 16;
  }
  const int ws_lds = kSAt + 1024 + wc * 256 + r * 4, xs_lds = kSAt + (wr * MT * 32 + r) * 4;
  constexpr int H0 = (MT + 1) / 2, H1 = MT / 2;
  i32x8 wf[2][2], x0[H0], x1[H1 > 0 ? H1 : 1];
  int bw[2], bx[MT];                               // the block's scales
  int place = 0;
  // Every step sends the same loads, past the end too (the last step once more, into places that nobody reads any more): the waits count
  // them, and there is no branch in the loop.  (With branches around them the products of two steps ended up behind the loads: 256 registers, spilled.)
  auto arrive = [&](auto half_tag) {               // the next step is in LDS, and everyone has read the one before
    constexpr int hh = decltype(half_tag)::value;
    if constexpr (STAGED) {
      if (hh == 1) return;
      lds_loads_wait<XL + 5>();                    // a stage behind this one's loads
    } else {
      lds_loads_wait<hh == 0 ? 4 : 5 + XL>();      // two steps of weights and, in a stage's second step, the next stage's rows and scales
    }
    __syncthreads();
  };
  auto send = [&](int s, auto half_tag) {          // the loads that take the place of step s - 1, or of the stage before
    constexpr int hh = decltype(half_tag)::value;
    const int u = s >> 1;
    if constexpr (hh == 0) load_s(u >> 2, (u & 3) == 0);
    if constexpr (STAGED) {
      if constexpr (hh == 0) {
        const int c = u + RS - 1, to = place == 0 ? RS - 1 : place - 1;
        load_x(c, to);
        load_w(2 * c, 2 * to);
        load_w(2 * c + 1, 2 * to + 1);
      }
    } else {
      if constexpr (hh == 0) load_x(u + 1, place ^ 1);
      load_w(s + 3, (s + 3) & 3);
    }
  };
  auto operand = [&](int a, int b) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(smem + a), hi = *reinterpret_cast<const i32x4*>(smem + b);
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto read_first = [&](auto half_tag) {
    constexpr int hh = decltype(half_tag)::value;
#pragma unroll
    for (int t = 0; t < 2; ++t) wf[hh][t] = operand(w_lds[hh] + t * 2048, w_lds[hh] + t * 2048 + 1024);
#pragma unroll
    for (int m = 0; m < H0; ++m) x0[m] = operand(x_lds[hh][0] + m * 4096, x_lds[hh][1] + m * 4096);
  };
  auto in_turn = [&](auto reads_tag, auto products_tag) {
    constexpr int R = decltype(reads_tag)::value, P = decltype(products_tag)::value, kEach = R > 0 && P > 0 ? (R + P - 1) / P : 1;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    }
  };
  auto step = [&](int s, auto half_tag, auto last_tag) {
    constexpr int hh = decltype(half_tag)::value;
    constexpr bool last = decltype(last_tag)::value;
    if constexpr (hh == 0) {
      const int at = (s >> 1 & 3) + (s >> 3 & 1) * 2048;
#pragma unroll
      for (int t = 0; t < 2; ++t) bw[t] = smem[ws_lds + t * 128 + at];
#pragma unroll
      for (int m = 0; m < MT; ++m) bx[m] = smem[xs_lds + m * 128 + at];
    }
#pragma unroll
    for (int m = 0; m < H1; ++m) x1[m] = operand(x_lds[hh][0] + (H0 + m) * 4096, x_lds[hh][1] + (H0 + m) * 4096);
    auto row_products = [&](const i32x8& rows, int m) {
#pragma unroll
      for (int t = 0; t < 2; ++t) acc[t][m] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[hh][t], rows, acc[t][m], 0, 0, 0, bw[t], 0, bx[m]);
    };
#pragma unroll
    for (int m = 0; m < H0; ++m) row_products(x0[m], m);
    in_turn(std::integral_constant<int, 2 * H1>{}, std::integral_constant<int, 2 * H0>{});
    if constexpr (hh == 1) {
      const int turn = place == RS - 1 ? 1 - RS : 1;
      place += turn;
      w_lds[0] += turn * 2 * kWStep;
      w_lds[1] += turn * 2 * kWStep;
#pragma unroll
      for (int i = 0; i < 4; ++i) x_lds[i / 2][i % 2] += turn * kXStage;
    }
    if constexpr (!last) {
      __builtin_amdgcn_sched_barrier(0);           // products of the first half stay ahead of the barrier, those of the other behind it
      arrive(std::integral_constant<int, hh ^ 1>{});
      __builtin_amdgcn_sched_barrier(0);
      read_first(std::integral_constant<int, hh ^ 1>{});
    }
    constexpr int kBefore = H1 / 2;
#pragma unroll
    for (int m = 0; m < kBefore; ++m) row_products(x1[m], H0 + m);
    if constexpr (!last) {
      in_turn(std::integral_constant<int, 4 + 2 * H0>{}, std::integral_constant<int, kBefore * 2>{});
      __builtin_amdgcn_sched_barrier(0);
      send(s + 1, std::integral_constant<int, hh ^ 1>{});
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int m = kBefore; m < H1; ++m) row_products(x1[m], H0 + m);
  };
  using Half0 = std::integral_constant<int, 0>;
  using Half1 = std::integral_constant<int, 1>;
  lds_loads_wait<0>();
  __syncthreads();
  send(0, Half0{});
  read_first(Half0{});
  for (int u = 0; u + 1 < p.U; ++u) {
    step(2 * u, Half0{}, std::false_type{});
    step(2 * u + 1, Half1{}, std::false_type{});
  }
  step(steps - 2, Half0{}, std::false_type{});
  step(steps - 1, Half1{}, std::true_type{});
  lds_loads_wait<0>();
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
         (long long)p.w_rows * p.U < 0x7fffffffLL && !(((uintptr_t)p.x | (uintptr_t)p.w) & 15) && (p.offsets || p.groups == 1) &&
         (!p.a_rows || (long long)x_rows * p.U * kF8Block <= 0xffffffffLL) && (long long)p.U * kF8TileBytes <= 0x7fffffffLL;
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
  const F8Tiles p{(const uint8_t*)x, (const uint8_t*)x_scales, (const uint8_t*)w_codes, (const uint8_t*)w_scales, f8_blocks(K), w_rows, a_rows, offsets, rows, groups, (uint32_t)((long long)x_rows * f8_blocks(K) * kF8Block), along, 0, 0};
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
  const F8Tiles p{(const uint8_t*)x, (const uint8_t*)x_scales, (const uint8_t*)w_codes, (const uint8_t*)w_scales, f8_blocks(K), w_rows, a_rows, offsets, rows, groups, (uint32_t)((long long)x_rows * f8_blocks(K) * kF8Block), along, 0, 0};
  if (!tiles_ok(p, x_rows)) return SHARPI_ERR_ARG;
  return launch_tiles<true>(p, F8Out{nullptr, (uint8_t*)codes, (uint8_t*)scales, score, I}, ga, height, stream);
}
