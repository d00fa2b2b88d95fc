// Products of many rows with weights in 8-bit floating point (fp8.h holds the format), in tiles on the scaled matrix instruction: one matrix, or
// the experts of a routing's sorted row list.  Two forms:
//   plain   out[row, :] = rows[row] W_e^T, bfloat16, or float where experts' outputs are still to be added up
//   gated   act(s g) (s u) with (g | u) the product, rounded to bfloat16 and quantised again: codes and scale bytes of the rows that the
//           second half of a feed-forward reads.  A block's 128 output columns are one block of the format, so the epilogue has what
//           it needs, and neither (g | u) nor the unquantised rows go to memory.
// Every output is one chain over k in ascending order (of each share of it): a row's result does not depend on which rows share its tile.
//
// Bound: 8,192 x 16,384 x 5,120 takes 547 us at best, 2.5 PFLOP/s, and 597 in a run of many (2.3): power takes the clock from 2.4 down to 1.5 to 1.7 GHz, of which the matrix
// cores are busy 73 %.  A loop of that instruction on registers alone runs at 4.8 PFLOP/s; the library's product in 8 bits (one scale a tensor) at 3.0 at 8,192 x 8,192 x
// 8,192, busy 90 % at 1.70 GHz, where these tiles are busy 77 % at 1.50: what is left to gain are waits, and power spent beside the products.
// Experts of few rows are bound by reading their weights: 16 of 2 x 8,192 x 5,120 with 6 rows each and one always on, 249 us, 5.7 TB/s.  With more rows the products'
// power and the memory's add up: a step of a tile of 16, 64, 128 and 256 rows over 5,120 takes 0.73, 0.88, 1.02 and 1.35 us with weights from memory, of 256 rows
// with weights in the caches 0.88 (16 experts with 128 rows each 364 us, 3.7 TB/s; the clock is at 2.0 GHz, the matrix cores busy 38 %).  Blocks that begin at places of k of their own: no change.
// Weights straight into registers instead of through LDS: 600 us for the first product above, then at 579.
#include <type_traits>

#include "fp8.h"
#include "lds_loads.h"

namespace {

constexpr int TW = 8;                  // waves a block: 2 along the rows x 4 along the columns
constexpr int TWC = 4;
constexpr int columns_of(int nt) { return 32 * nt * TWC; }      // weight rows of a block: nt tiles of 32 a column wave
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
  int height;                // rows of a tile at most, a multiple of 64
  int tiles, nb;             // row tiles in all at most; column blocks
  int shares;                // of the blocks of k (plain form): share s of them gives row s * rows + row of the result
};

// plain: out [rows, n_out], bfloat16 or float.  gated: codes [rows, 128 f8_blocks(n_out)], scales [rows, f8_scale_stride(n_out)], score [rows] or null.
struct F8Out {
  void* out;
  uint8_t* codes;
  uint8_t* scales;
  const float* score;
  int n_out;
};

// Where 16-byte piece `piece` of row `row` of a step is kept: the pieces that sixteen neighbouring lanes read fall into the sixteen 16-byte groups
// of the banks.
__device__ __forceinline__ int row_piece(int row, int piece) { return piece ^ ((row >> 2) & 3); }

// Two kernels.  PAIRED: tiles of up to 128 rows, two blocks a compute unit, which fill each other's gaps (a tile's first loads, its barriers, its
// end); the other: tiles of up to 256, one block a unit, for what many rows share.
// The paired kernels spill up to four vector registers, the gated tall one scalar ones only.
// (us, paired and not: 64 experts of 2 x 1,408 x 2,048, 94 rows each 108 and 119; 16 of 16,384 x 5,120, 128 rows each 383 and 364.)
// LDS holds a ring of slots, a slot one step (64 of k: 16 KB of weights, 4 KB of rows for each MT), or two steps of low tiles in a block of its own,
// whose steps are short beside a barrier.
constexpr int step_bytes(int mt, int nt) { return 8192 * nt + 4096 * mt; }
template <bool PAIRED> struct Ring {
  static constexpr int kHighest = PAIRED ? 2 : 4;                       // a tile has up to 64 x this many rows
  static constexpr int steps(int mt) { return !PAIRED && mt <= 2 ? 2 : 1; }
  static constexpr int slots(int mt) { return PAIRED || mt <= 2 ? 3 : 4; }
  static constexpr int scales_at(int mt) { return slots(mt) * steps(mt) * step_bytes(mt, 2); }
  static constexpr int kRowScales = 256 * kHighest, kChunk = kRowScales + 1024;       // bytes of a chunk's scales: rows', then weights'
  static constexpr int kLds = scales_at(2) + 3 * kChunk;
  static_assert(scales_at(1) <= scales_at(2) && (PAIRED || (scales_at(3) <= scales_at(2) && scales_at(4) <= scales_at(2))), "the largest ring");
};

// Gated results near a border of two codes.  The instruction's products are off by some 2e-5 of a sum's rms (fp8.h), now and then by ten times that, which moves 1
// value in 390 across a border of e4m3 (float sums 1 in 170,000 and fewer), a sixteenth to an eighth of it: nearly as much error in the layer's result as that result's
// rounding to bfloat16.  Values h that kNear |h| / top of them would move, if they are at least 1 / kNearTop of their block's largest, top (they carry most of the
// error), are computed once more in float from their rows of codes: about 5 of a tile of 256 x 128, in 4 to 8 us of a tile's 30 to 80 (3,001 rows through
// 2 x 2,816 x 2,048 57 -> 65 us, 2,048 through 16 experts of 2 x 8,192 x 5,120 and one always on 522 -> 585).  Of these large values 1 in 24,000 or fewer is then off, for 1 in 3,000.  Over
// 1,400 drawn sizes the layer's error against 64 bits is 1.11 times that of the same sums in float (1.40 at most), without this 1.34 (3.6).  The list has room for all of a tile's values, behind its codes in the ring: a row's
// codes are the same alone, again and again in one tile, and beside any others.  The whole product on the bfloat16 instruction would take twice the matrix cores' time.
constexpr float kNear = 1.5e-4f;
constexpr float kNearTop = 4.f;
// Of more than kNearMany values kNearRows neighbours of the list go together where they are of one column, whose pieces lie in lines of their own and take longer than the rows': equal rows
// have all of their values near a border in the same columns.  (2,048 equal rows through 2 x 8,192 x 5,120 and back, in the order of their values near a border: 315 to 420 us, by one at a
// time 412 to 554, where rows that differ take 265; 3,001 through 2 x 2,816 x 2,048 81 to 108, 80 to 142 and 95.)
constexpr int kNearMany = 64, kNearRows = 4;
// Two columns' products of ROWS rows in float, dealt to the wave: x: a row's codes and scales; w: a column's first piece in its tile, ws: its scales.  A lane's
// pieces come in their order, whatever ROWS and kFlight (pieces on their way at a time) are, so every row gets the same sum.
struct F8Source {
  const uint8_t* codes;
  const uint8_t* scales;
};
template <int kFlight, int ROWS>
__device__ __forceinline__ void f8_row_dots(const F8Source (&x)[ROWS], const F8Source (&w)[2], int U, float2 (&out)[ROWS]) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  const int lane = threadIdx.x & (kWave - 1), pieces = U * 8;
  float sum[ROWS][2];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) sum[r][0] = sum[r][1] = 0.f;
  for (int p0 = lane; p0 < pieces; p0 += kFlight * kWave) {
    i32x4 xv[ROWS][kFlight], wv[2][kFlight];
    int xb[ROWS][kFlight], wb[2][kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int q = min(p0 + i * kWave, pieces - 1), u = q >> 3, j = q & 7;       // piece j of a block: k = 16 j
      const size_t at = (size_t)u * kF8TileBytes + (j >> 2) * 2048 + (j & 1) * 1024 + (j >> 1 & 1) * 512;
      const int byte = (u >> 2) * 128 + (u & 3);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        xv[r][i] = *reinterpret_cast<const i32x4*>(x[r].codes + (size_t)q * 16);
        xb[r][i] = x[r].scales[u];
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        wv[t][i] = *reinterpret_cast<const i32x4*>(w[t].codes + at);
        wb[t][i] = w[t].scales[byte];
      }
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      if (p0 + i * kWave >= pieces) continue;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(xv[r][i][c], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(xv[r][i][c], true);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const f32x2 d = __builtin_amdgcn_cvt_pk_f32_fp8(wv[t][i][c], false), f = __builtin_amdgcn_cvt_pk_f32_fp8(wv[t][i][c], true);
            s[t] = fmaf(a[0], d[0], s[t]);
            s[t] = fmaf(a[1], d[1], s[t]);
            s[t] = fmaf(b[0], f[0], s[t]);
            s[t] = fmaf(b[1], f[1], s[t]);
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) sum[r][t] += f8_scaled(s[t], xb[r][i] + wb[t][i]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) out[r] = make_float2(wave_sum(sum[r][0]), wave_sum(sum[r][1]));
}

// One tile: rows row0 .. row_end (up to 64 MT of them) of matrix e against column block nblock.  MT: groups of 32 rows a wave; NT: weight tiles of a wave.
template <int MT, int NT, bool GATED, bool PAIRED, typename TO>
__device__ __forceinline__ void f8_tile(const F8Tiles& p, const F8Out& o, GatedAct act, int e, int row0, int row_end, int nblock, unsigned char* smem,
                                        float (*s_top)[64 * Ring<PAIRED>::kHighest], int* n_near) {
  using RG = Ring<PAIRED>;
  constexpr int NS = RG::steps(MT), RING = RG::slots(MT) * NS, AHEAD = RING - NS;      // (steps)
  static_assert(NT == 2 || !GATED, "a gated tile's columns are a block of the format");
  constexpr int kTileCols = columns_of(NT), kWStep = 8192 * NT, kStep = step_bytes(MT, NT), kSAt = RG::scales_at(MT);
  const int lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, g = lane >> 5;
  const int wr = wid / TWC, wc = wid % TWC;
  const bool sorted = row0 < p.rows;             // of the sorted list, not of the rows behind it
  const int U4 = (p.U + 3) >> 2;
  const int half = p.w_rows / 64;                // gated: tiles of the gate rows
  const bool exists = !GATED || nblock * (kTileCols / 64) + wc < half;
  // Loads go straight into LDS.  Weights: wave wid brings tile wid of the block's eight (gated: a wave column's gate tile, then its up tile), a step is
  // 2 KB of it on end; of four tiles half a step each.  Rows: a load brings 16 rows of 64 bytes, their 16-byte pieces exchanged by row bits (row_piece).  Rows behind the last read it
  // again; what they give is never stored.  Scales: a chunk of four blocks of k is a word a row; waves 0 to 3 bring those of 64 rows each,
  // waves 4 to 7 those of two weight tiles each.
  auto block_tile = [&](int lt) {
    if constexpr (GATED) return min(nblock * (kTileCols / 64) + lt / 2, half - 1) + lt % 2 * half;
    else return min(nblock * (kTileCols / 32) + lt, p.w_rows / 32 - 1);
  };
  const size_t w_at = (size_t)e * (p.w_rows / 32);
  const u32x4 wb = buffer_of(p.w + (w_at + block_tile(NT == 2 ? wid : wid >> 1)) * p.U * kF8TileBytes, (uint32_t)p.U * kF8TileBytes);
  const uint32_t lds0 = lds_address((const char*)smem);
  const uint32_t x_stride = (uint32_t)p.U * kF8Block;
  const size_t x_first = p.a_rows ? 0 : row0;             // (rows in a row: the tile's own piece of x, at any distance)
  const uint32_t x_bytes = p.a_rows ? p.x_bytes : (uint32_t)(row_end - row0) * x_stride;
  const u32x4 xb = buffer_of(p.x + x_first * x_stride, x_bytes);
  auto x_row = [&](int lrow) {
    const int row = min(row0 + lrow, row_end - 1);
    return !p.a_rows ? row - row0 : sorted ? p.a_rows[row] : row - p.rows;
  };
  constexpr int XL = (MT + 1) / 2;                        // loads of rows a wave and step (of 4 MT; some twice, to the same place)
  // this block's steps of k (a share: whole blocks)
  const int first_step = 2 * (int)((long long)p.U * blockIdx.y / gridDim.y), steps = 2 * (int)((long long)p.U * (blockIdx.y + 1) / gridDim.y);
  const uint32_t w_off[2] = {(uint32_t)lane * 16 + (NT == 1 ? (wid & 1) * 1024 : 0), (uint32_t)lane * 16 + 1024};
  auto load_w = [&](int s, uint32_t at) {                 // (past the end: the last step once more, for nobody)
    const uint32_t from = min(s, steps - 1) * 2048, to = lds0 + at + wid * (1024 * NT);
    if constexpr (NT == 2) load_two_to_lds<false>(wb, w_off[0], w_off[1], from, to, to + 1024);
    else load_to_lds<false>(wb, w_off[0], from, to);
  };
  uint32_t x_off[XL], xs_off;
  int x_to[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int li = (wid * XL + i) % (4 * MT), lrow = li * 16 + (lane >> 2);
    x_to[i] = kWStep + li * 1024;
    x_off[i] = (uint32_t)x_row(lrow) * x_stride + row_piece(lrow, lane & 3) * 16;
  }
  // scales: the wave's own buffer
  u32x4 sb;
  if (wid < 4) {
    const int lrow = min(wid, MT - 1) * 64 + lane;
    xs_off = (uint32_t)x_row(lrow) * (U4 * 4);
    sb = buffer_of(p.xs + x_first * (U4 * 4), p.a_rows ? (uint32_t)(p.x_bytes / x_stride) * (U4 * 4) : (uint32_t)(row_end - row0) * (U4 * 4));
  } else {
    const int lt = (wid - 4) * 2 % (4 * NT);              // (of four tiles twice, to the same place)
    const int t0 = block_tile(lt), t1 = block_tile(lt + 1);
    const uint8_t* base = p.ws + w_at * U4 * 128;
    const int low = min(t0, t1);                          // (the descriptor begins at the lower of the two tiles)
    xs_off = (uint32_t)((lane < 32 ? t0 : t1) - low) * (U4 * 128) + (lane & 31) * 4;
    sb = buffer_of(base + (size_t)low * U4 * 128, (uint32_t)(max(t0, t1) - low + 1) * (U4 * 128));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sb[i] = (uint32_t)__builtin_amdgcn_readfirstlane(sb[i]);
  const uint32_t s_lds = lds0 + kSAt + (wid < 4 ? min(wid, MT - 1) * 256 : RG::kRowScales + (wid - 4) % (2 * NT) * 256);
  const uint32_t s_step = wid < 4 ? 4 : 128;
  // waited for here: the compiler's own waits must not fall among the loads below, which it does not know of
#pragma unroll
  for (int i = 0; i < XL; ++i) asm volatile("" : "+v"(x_off[i]));
  asm volatile("" : "+v"(xs_off));
  // the scales of the chunk behind chunk c, once a chunk; the other blocks' loads go where nobody reads
  auto load_s = [&](int c, bool first) { load_words_to_lds(sb, xs_off, min(c + 1, U4 - 1) * s_step, s_lds + (first ? ((c + 1) & 1) : 2) * RG::kChunk); };
  auto load_x = [&](int s, uint32_t at) {
    uint32_t to[XL];
#pragma unroll
    for (int i = 0; i < XL; ++i) to[i] = lds0 + at + x_to[i];
    bring_all_to_lds<true, XL>(xb, x_off, min(s, steps - 1) * 64, to);
  };
  load_s((first_step >> 3) - 1, true);
  load_s(first_step >> 3, true);                          // (the next chunk may begin a block further on)
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) {
    load_w(first_step + s, s * kStep);
    load_x(first_step + s, s * kStep);
  }

  f32x16 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][m][i] = 0.f;
  // operand addresses: W of the step, and piece q of a lane's 32 bytes of its rows
  int w_lds = wc * (2048 * NT) + lane * 16, x_lds[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) x_lds[q] = kWStep + (wr * MT * 32 + r) * 64 + row_piece(r, g * 2 + q) * 16;
  const int ws_lds = kSAt + RG::kRowScales + wc * (128 * NT) + r * 4, xs_lds = kSAt + (wr * MT * 32 + r) * 4;
  constexpr int H0 = (MT + 1) / 2, H1 = MT / 2;
  i32x8 wf[NT], x0[H0], x1[H1 > 0 ? H1 : 1];
  int bw[NT], bx[MT];                               // the block's scales
  auto operand = [&](int a, int b) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(smem + a), hi = *reinterpret_cast<const i32x4*>(smem + b);
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto read_w = [&](i32x8 (&to)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) to[t] = operand(w_lds + t * 2048, w_lds + t * 2048 + 1024);
  };
  auto read_rows = [&](i32x8* to, int m0, int n) {
#pragma unroll
    for (int m = 0; m < n; ++m) to[m] = operand(x_lds[0] + (m0 + m) * 2048, x_lds[1] + (m0 + m) * 2048);
  };
  auto read_scales = [&](int u, int (&w)[NT], int (&x)[MT]) {
    const int at = (u & 3) + (u >> 2 & 1) * RG::kChunk;
#pragma unroll
    for (int t = 0; t < NT; ++t) w[t] = smem[ws_lds + t * 128 + at];
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = smem[xs_lds + m * 128 + at];
  };
  int at = 0;                                      // this step's bytes in the ring
  auto ahead = [&](int n) {                        // those of n steps on
    const int a = at + n * kStep;
    return (uint32_t)(a >= RING * kStep ? a - RING * kStep : a);
  };
  // A step.  Its weights and first row groups are in registers; it reads the others while the first are multiplied, and the next step's
  // first part, behind the barrier, while the others are.  The loads AHEAD steps on go out one by one among the products (a wave that
  // sends all of a stage's on end stands still until the memory pipe has taken them).  Every step sends the same loads, so that the waits
  // count them and the loop has no branch (with branches around them the products of two steps ended up behind the loads: 256 registers, spilled).
  auto step = [&](int s, auto half_tag) {
    constexpr int hh = decltype(half_tag)::value;
    auto row_products = [&](const i32x8& rows, int m) {
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][m] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[t], rows, acc[t][m], 0, 0, 0, bw[t], 0, bx[m]);
    };
    if constexpr (H1 > 0) read_rows(x1, H0, H1);
    row_products(x0[0], 0);
    __builtin_amdgcn_sched_barrier(0);
    load_x(s + AHEAD, ahead(AHEAD));
    if constexpr (hh == 0) load_s(s >> 3, (s & 6) == 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 1; m < H0; ++m) row_products(x0[m], m);
    __builtin_amdgcn_sched_barrier(0);             // products of the first row groups stay ahead of the barrier, those of the others behind it
    if constexpr (NS == 1 || hh == 1) {
      // the next slot is here, and everyone has read the one before: counted are the slots behind it (a scales' load among them makes the wait one longer)
      lds_loads_wait<(AHEAD - NS) * (NT + XL)>();
      __syncthreads();
    }
    const int turn = at == (RING - 1) * kStep ? (1 - RING) * kStep : kStep;
    at += turn;
    w_lds += turn;
    x_lds[0] += turn;
    x_lds[1] += turn;
    __builtin_amdgcn_sched_barrier(0);
    i32x8 wn[NT];
    int nw[NT], nx[MT];
    if constexpr (hh == 1) read_scales((s + 1) >> 1, nw, nx);
    read_w(wn);
    read_rows(x0, 0, H0);
    if constexpr (H1 > 0) row_products(x1[0], H0);
    __builtin_amdgcn_sched_barrier(0);
    load_w(s + 1 + AHEAD, ahead(AHEAD));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 1; m < H1; ++m) row_products(x1[m], H0 + m);
#pragma unroll
    for (int t = 0; t < NT; ++t) wf[t] = wn[t];
    if constexpr (hh == 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t) bw[t] = nw[t];
#pragma unroll
      for (int m = 0; m < MT; ++m) bx[m] = nx[m];
    }
  };
  lds_loads_wait<0>();
  __syncthreads();
  read_scales(first_step >> 1, bw, bx);
  read_w(wf);
  read_rows(x0, 0, H0);
  load_w(first_step + AHEAD, AHEAD * kStep);
  for (int s = first_step; s < steps; s += 2) {
    step(s, std::integral_constant<int, 0>{});
    step(s + 1, std::integral_constant<int, 1>{});
  }
  lds_loads_wait<0>();
  // a lane holds, of row row0 + (wr MT + m) 32 + r, columns 8 q + 4 g + 0..3 (q 0..3) of tile t
  if constexpr (!GATED) {
    const int n_base = nblock * kTileCols + wc * (32 * NT);
    if (n_base >= o.n_out) return;
    // The results go through the wave's own part of LDS (everyone has read the last step), a row group at a time, to leave as whole lines of 64 NT bytes;
    // a lane first exchanges halves with lane ^ 32, so that it has eight columns of its row.  Rows that do not begin at 16-byte addresses are
    // stored by elements.  (Stored from the registers, pieces of 16 bytes a row, 8,192 x 2,048 x 2,560 in one round of tiles took 49 us, so 39.)
    constexpr int V = 16 / sizeof(TO), P = 32 * NT / V;      // columns of a 16-byte piece, pieces of a row
    TO* out = (TO*)o.out + (size_t)blockIdx.y * p.rows * o.n_out;
    const bool wide = o.n_out % V == 0 && ((uintptr_t)o.out & 15) == 0;
    __syncthreads();
    unsigned char* mine = smem + wid * (32 * P * 16);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int first = row0 + (wr * MT + m) * 32;
      if (first >= row_end) break;                  // (the wave's)
      if (wide) {
        auto keep = [&](int piece, const uint4& v) { *reinterpret_cast<uint4*>(mine + r * (P * 16) + (piece ^ (r & (P < 8 ? P - 1 : 7))) * 16) = v; };
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const f32x16& v = acc[t][m];
          if constexpr (sizeof(TO) == 4) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              keep(t * 8 + q * 2 + g, make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3])));
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const auto lo = __builtin_amdgcn_permlane32_swap(f32_to_bf16_pair(v[8 * h], v[8 * h + 1]), f32_to_bf16_pair(v[8 * h + 4], v[8 * h + 5]), false, false);
              const auto hi = __builtin_amdgcn_permlane32_swap(f32_to_bf16_pair(v[8 * h + 2], v[8 * h + 3]), f32_to_bf16_pair(v[8 * h + 6], v[8 * h + 7]), false, false);
              keep(t * 4 + h * 2 + g, make_uint4(lo[0], hi[0], lo[1], hi[1]));
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 32 * P / kWave; ++i) {
          const int lrow = i * (kWave / P) + lane / P, n = n_base + lane % P * V;
          const uint4 v = *reinterpret_cast<const uint4*>(mine + lrow * (P * 16) + (lane % P ^ (lrow & (P < 8 ? P - 1 : 7))) * 16);
          if (first + lrow < row_end && n < o.n_out) *reinterpret_cast<uint4*>(out + (size_t)(first + lrow) * o.n_out + n) = v;
        }
      } else if (first + r < row_end) {
        TO* dst = out + (size_t)(first + r) * o.n_out;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int n = n_base + t * 32 + (i / 4) * 8 + g * 4 + i % 4;
            if (n < o.n_out) dst[n] = from_f32<TO>(acc[t][m][i]);
          }
      }
    }
  } else {
    const int U2 = f8_blocks(o.n_out), su2 = f8_scale_stride(o.n_out);
    float h[MT][16];
    bool bad = false;                              // (a value of the lane's is not finite)
    // the values near a border, each row << 7 | column of the tile, behind the codes
    static_assert(64 * MT * kF8Block * 3 <= RG::slots(MT) * NS * kStep, "codes and a list of all of them fit in the ring");
    unsigned short* near = reinterpret_cast<unsigned short*>(smem + 64 * MT * kF8Block);
    auto units = [&](auto code_tag) {              // (the activation is chosen once a tile)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int lrow = (wr * MT + m) * 32 + r, row = min(row0 + lrow, row_end - 1);
        const float sc = o.score != nullptr && sorted ? o.score[row] : 1.f;
        uint32_t top = 0, all = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float v = exists ? f8_unit<decltype(code_tag)::value>(act.limit, acc[0][m][i] * sc, acc[1][m][i] * sc) : 0.f;
          const uint32_t b = __float_as_uint(bf16_to_f32(f32_to_bf16(v))) & 0x7fffffffu;
          if (b < 0x7f800000u && b > top) top = b;
          all = b > all ? b : all;
          h[m][i] = v;
        }
        bad = bad || all >= 0x7f800000u;
        const float t2 = reduce32(__uint_as_float(top), MaxOf{});
        if (g == 0) s_top[wc][lrow] = t2;
      }
    };
    if (act.code == ACT_SWISH_CLAMP) units(std::integral_constant<int, ACT_SWISH_CLAMP>{});
    else if (act.code == ACT_GELU_TANH) units(std::integral_constant<int, ACT_GELU_TANH>{});
    else units(std::integral_constant<int, ACT_SILU>{});
    if (threadIdx.x == 0) *n_near = 0;
    __syncthreads();
    // the codes through LDS, to leave as whole lines: a row's 128 are one block of the format
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int lrow = (wr * MT + m) * 32 + r;
      const float t = fmaxf(fmaxf(s_top[0][lrow], s_top[1][lrow]), fmaxf(s_top[2][lrow], s_top[3][lrow]));
      const int s = f8_scale_of(__float_as_uint(t));
      const float scale = f8_scale_value(s), by = t > 0.f ? kNear / t : 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        auto codes_of = [&](float by) {
          auto moved = [&](int i) { return fmaf(h[m][4 * q + i], fabsf(h[m][4 * q + i]) * by, h[m][4 * q + i]); };
          return f8_codes4(f32_to_bf16_pair(moved(0), moved(1)), f32_to_bf16_pair(moved(2), moved(3)), scale);
        };
        uint32_t c = codes_of(-by);
        if (const uint32_t differ = c ^ codes_of(by)) {
          c = codes_of(0.f);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (const float a = fabsf(h[m][4 * q + i]); (differ >> (8 * i) & 0xff) && a * kNearTop >= t && a <= t * 1.01f && row0 + lrow < row_end)
              near[atomicAdd(n_near, 1)] = (unsigned short)(lrow << 7 | (wc * 32 + q * 8 + g * 4 + i));
        }
        if (bad)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((__float_as_uint(bf16_to_f32(f32_to_bf16(h[m][4 * q + i]))) & 0x7f800000u) == 0x7f800000u) c |= kF8Nan << (8 * i);
        *reinterpret_cast<uint32_t*>(smem + lrow * 128 + ((wc * 2 + (q >> 1)) ^ (lrow & 7)) * 16 + (q & 1) * 8 + g * 4) = c;
      }
      if (wc == 0 && g == 0 && row0 + lrow < row_end) o.scales[(size_t)(row0 + lrow) * su2 + nblock] = (uint8_t)s;
    }
    __syncthreads();
    const int total = __builtin_amdgcn_readfirstlane(*n_near);
    // values of one column, computed again and put in their places
    auto again = [&](auto flight_tag, auto rows_tag, const int (&lrow)[decltype(rows_tag)::value], int column) {
      constexpr int N = decltype(rows_tag)::value;
      auto source = [&](int which) {
        const size_t at = w_at + block_tile(2 * (column >> 5) + which);
        return F8Source{p.w + at * p.U * kF8TileBytes + (column & 31) * 16, p.ws + at * U4 * 128 + (column & 31) * 4};
      };
      const F8Source w[2] = {source(0), source(1)};
      F8Source x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const size_t x_at = x_first + __builtin_amdgcn_readfirstlane(x_row(lrow[j]));
        x[j] = {p.x + x_at * x_stride, p.xs + x_at * (U4 * 4)};
      }
      float2 v[N];
      f8_row_dots<decltype(flight_tag)::value, N>(x, w, p.U, v);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float sc = o.score != nullptr && sorted ? o.score[row0 + lrow[j]] : 1.f;
        const float t = fmaxf(fmaxf(s_top[0][lrow[j]], s_top[1][lrow[j]]), fmaxf(s_top[2][lrow[j]], s_top[3][lrow[j]]));
        const uint32_t pair = f32_to_bf16_pair(f8_unit(act, v[j].x * sc, v[j].y * sc), 0.f);
        const uint32_t c = (pair & 0x7f80u) == 0x7f80u ? kF8Nan : f8_codes4(pair, 0u, f8_scale_value(f8_scale_of(__float_as_uint(t))));
        if (lane == 0) smem[lrow[j] * 128 + ((column >> 4) ^ (lrow[j] & 7)) * 16 + (column & 15)] = (unsigned char)c;
      }
    };
    const bool many = total > kNearMany;
    for (int i = many ? wid * kNearRows : wid; i < total; i += many ? TW * kNearRows : TW) {
      int left = 1;
      if (many) {
        left = min(kNearRows, total - i);
        int lrow[kNearRows];
        const int column = __builtin_amdgcn_readfirstlane(near[i]) & 127;
        bool same = left == kNearRows;
#pragma unroll
        for (int j = 0; j < kNearRows; ++j) {
          const int entry = __builtin_amdgcn_readfirstlane(near[min(i + j, total - 1)]);
          lrow[j] = entry >> 7;
          same = same && (entry & 127) == column;
        }
        if (same) {
          again(std::integral_constant<int, 1>{}, std::integral_constant<int, kNearRows>{}, lrow, column);
          left = 0;
        }
      }
#pragma unroll 1
      for (int j = 0; j < left; ++j) {
        const int entry = __builtin_amdgcn_readfirstlane(near[i + j]), one[1] = {entry >> 7};
        again(std::integral_constant<int, PAIRED ? 3 : 6>{}, std::integral_constant<int, 1>{}, one, entry & 127);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int lrow = (wid * MT + i) * 8 + (lane >> 3), row = row0 + lrow;
      const uint4 v = *reinterpret_cast<const uint4*>(smem + lrow * 128 + ((lane & 7) ^ (lrow & 7)) * 16);
      if (row < row_end) *reinterpret_cast<uint4*>(o.codes + ((size_t)row * U2 + nblock) * kF8Block + (lane & 7) * 16) = v;
    }
  }
}

// The order of the tiles: row tile by row tile, the column blocks of a row tile side by side (64 at a time).  Blocks go to the dies round-robin, so a die
// keeps its column blocks and its L2 their weights from one row tile to the next, and all of the chip is in the same few row tiles.
constexpr int kSideBySide = 64;

template <int NT, bool GATED, bool PAIRED, typename TO = bf16_t>
__global__ __launch_bounds__(TW* kWave, PAIRED ? 4 : 2) void fp8_tiles_kernel(F8Tiles p, F8Out o, GatedAct act) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[Ring<PAIRED>::kLds];
  __shared__ float s_top[GATED ? TWC : 1][64 * Ring<PAIRED>::kHighest];
  __shared__ int s_found[3];
  __shared__ int s_near;
  const int lane = threadIdx.x & (kWave - 1);
  const int slot = blockIdx.x;
  const int c0 = slot / (kSideBySide * p.tiles) * kSideBySide, left = slot - c0 * p.tiles, wide = min(kSideBySide, p.nb - c0);
  int tile = left / wide;
  const int nblock = c0 + left % wide;
  // the rows behind the list, whose tiles are bound by products and take long, go evenly among the first half of the experts', which are bound by
  // reading their weights (16 experts of 8,192 x 5,120, 2,048 tokens and as many rows behind: 456 and 282 us; among all of them 492 and 287)
  const int along = p.along > 0 ? (p.along + p.height - 1) / p.height : 0;
  if (along) {
    const int spread = max(along, p.tiles / 2);
    const int before = min(along, (int)((long long)tile * along / spread));
    if (tile < spread && (int)((long long)(tile + 1) * along / spread) > before) tile = -1 - before;
    else tile -= before;
  }
  int e = 0, row0 = tile * p.height, row_end = min(p.rows, row0 + p.height);
  if (p.offsets) {
    // the groups' tiles are numbered through: as few of up to `height` rows as hold a group's, all of one height
    if (tile < 0) {
      const int n = along, each = ((p.along + n - 1) / n + 63) & ~63;
      e = p.groups;
      row0 = p.rows + (-1 - tile) * each;
      row_end = min(p.rows + p.along, row0 + each);
    } else {
      if (threadIdx.x < kWave) {
        int before = 0, found = -1, first_row = 0, last_row = 0;
        for (int c = 0; c < p.groups && found < 0; c += kWave) {
          const int i = c + lane;
          const int from = p.offsets[min(i, p.groups)], to = p.offsets[min(i + 1, p.groups)];
          const int mine = (to - from + p.height - 1) / p.height;
          int upto = mine;
#pragma unroll
          for (int k = 1; k < kWave; k <<= 1) {
            const int up = __shfl_up(upto, k, kWave);
            if (lane >= k) upto += up;
          }
          const int first = before + upto - mine;
          const unsigned long long here = __builtin_amdgcn_ballot_w64(mine > 0 && tile >= first && tile < first + mine);
          if (here) {
            const int l = __ffsll((long long)here) - 1;
            const int n = __shfl(mine, l, kWave), f = __shfl(from, l, kWave), t = __shfl(to, l, kWave);
            const int each = ((t - f + n - 1) / n + 63) & ~63;
            found = c + l;
            first_row = f + (tile - __shfl(first, l, kWave)) * each;
            last_row = min(t, first_row + each);
          }
          before += __shfl(upto, kWave - 1, kWave);
        }
        if (threadIdx.x == 0) {
          s_found[0] = found;
          s_found[1] = first_row;
          s_found[2] = last_row;
        }
      }
      __syncthreads();
      e = __builtin_amdgcn_readfirstlane(s_found[0]);
      row0 = __builtin_amdgcn_readfirstlane(s_found[1]);
      row_end = __builtin_amdgcn_readfirstlane(s_found[2]);
      if (e < 0) return;
    }
  }
  const int rows = row_end - row0;
  if (rows <= 0) return;
#define F8_TILE(MTV) f8_tile<MTV, NT, GATED, PAIRED, TO>(p, o, act, e, row0, row_end, nblock, smem, s_top, &s_near)
  if (rows <= 64) F8_TILE(1);
  else if (PAIRED || rows <= 128) F8_TILE(2);
  else if constexpr (!PAIRED) {
    if (rows <= 192) F8_TILE(3);
    else F8_TILE(4);
  }
#undef F8_TILE
}

bool tiles_ok(const F8Tiles& p, int x_rows) {
  return p.rows > 0 && x_rows > 0 && p.U > 0 && p.U <= f8_blocks(kF8MostK - 1) && p.w_rows > 0 && p.w_rows % kF8Tile == 0 && p.groups > 0 && p.groups < kMaxGroups &&
         p.along >= 0 && (p.offsets || !p.along) && (long long)p.rows + p.along <= 0x7fffff00LL && (long long)p.w_rows * p.U < 0x7fffffffLL &&
         !(((uintptr_t)p.x | (uintptr_t)p.w) & 15) && !(((uintptr_t)p.xs | (uintptr_t)p.ws) & 3) && (p.offsets || p.groups == 1) &&
         (!p.a_rows || (long long)x_rows * p.U * kF8Block <= 0xffffffffLL);
}

template <bool GATED> int launch_tiles(F8Tiles p, const F8Out& o, GatedAct act, int nt, int dtype, hipStream_t stream) {
  const int height = p.height;
  if (height < 64 || height > 64 * Ring<false>::kHighest || height % 64) return SHARPI_ERR_ARG;
  if (!p.a_rows && (long long)height * p.U * kF8Block > 0xffffffffLL) return SHARPI_ERR_ARG;      // (a tile's rows: one descriptor of its loads)
  const long long tiles = p.offsets ? (long long)p.rows / height + (p.rows < p.groups ? p.rows : p.groups) + (p.along + height - 1) / height
                                    : (p.rows + height - 1) / height;
  if ((nt != 1 && nt != 2) || (nt == 1 && (GATED || height <= 64 * Ring<true>::kHighest))) return SHARPI_ERR_ARG;
  p.nb = ceil_div(o.n_out, GATED ? columns_of(nt) / 2 : columns_of(nt));
  p.tiles = (int)tiles;
  if (tiles * p.nb > 0x7fffff) return SHARPI_ERR_ARG;        // (of 512 threads each, of which a launch has at most 2^32 along x)
  if (p.shares < 1 || p.shares > p.U || (p.shares > 1 && (GATED || p.offsets || dtype != DT_F32))) return SHARPI_ERR_ARG;
  const dim3 grid((unsigned)(tiles * p.nb), (unsigned)p.shares), block(TW * kWave);
  if constexpr (!GATED) {
    if (dtype == DT_F32) {
      if (height <= 64 * Ring<true>::kHighest) fp8_tiles_kernel<2, false, true, float><<<grid, block, 0, stream>>>(p, o, act);
      else if (nt == 1) fp8_tiles_kernel<1, false, false, float><<<grid, block, 0, stream>>>(p, o, act);
      else fp8_tiles_kernel<2, false, false, float><<<grid, block, 0, stream>>>(p, o, act);
      SHARPI_CHECK_LAUNCH();
      return SHARPI_OK;
    }
  }
  if (dtype != DT_BF16) return SHARPI_ERR_ARG;
  if (height <= 64 * Ring<true>::kHighest) fp8_tiles_kernel<2, GATED, true><<<grid, block, 0, stream>>>(p, o, act);
  else if (nt == 2) fp8_tiles_kernel<2, GATED, false><<<grid, block, 0, stream>>>(p, o, act);
  else if constexpr (!GATED) fp8_tiles_kernel<1, GATED, false><<<grid, block, 0, stream>>>(p, o, act);
  SHARPI_CHECK_LAUNCH();
  return SHARPI_OK;
}

}  // namespace

// out [rows, N], dtype DT_BF16 or DT_F32; with shares > 1 (DT_F32, one matrix) [shares, rows, N] to be added up.  x: codes [x_rows, 128 U] and scales; w_rows: stored rows of one matrix; a_rows, offsets: of a sorted row list, or null; along: rows
// behind the list's `rows`, which matrix `groups` takes (row i reads row i - rows of x if there is a_rows); height: rows of a tile at most (64, 128, 192, 256); nt: its columns, 128 nt (1 with heights from 192 on).
SHARPI_EXPORT int sharpi_fp8_tiles(const void* x, const void* x_scales, int x_rows, const void* w_codes, const void* w_scales, int w_rows, void* out, int dtype,
                                   int rows, int N, int K, const int* a_rows, const int* offsets, int groups, int along, int height, int nt, int shares,
                                   hipStream_t stream) {
  if (rows <= 0) return SHARPI_OK;
  if (N <= 0 || K <= 0 || w_rows != f8_padded_rows(N)) return SHARPI_ERR_ARG;
  const F8Tiles p{(const uint8_t*)x, (const uint8_t*)x_scales, (const uint8_t*)w_codes, (const uint8_t*)w_scales, f8_blocks(K), w_rows, a_rows, offsets, rows, groups, (uint32_t)((long long)x_rows * f8_blocks(K) * kF8Block), along, height, 0, 0, shares};
  if (!tiles_ok(p, x_rows)) return SHARPI_ERR_ARG;
  return launch_tiles<false>(p, F8Out{out, nullptr, nullptr, nullptr, N}, GatedAct{}, nt, dtype, stream);
}

// codes [rows, 128 f8_blocks(I)] and scales [rows, f8_scale_stride(I)] of act(s g) (s u); w_rows: twice I up to a multiple of 32; score [rows] or null.
SHARPI_EXPORT int sharpi_fp8_tiles_gated(const void* x, const void* x_scales, int x_rows, const void* w_codes, const void* w_scales, int w_rows,
                                         void* codes, void* scales, int rows, int I, int K, const int* a_rows, const int* offsets, int groups, int along,
                                         const float* score, int act, float limit, int height, hipStream_t stream) {
  if (rows <= 0) return SHARPI_OK;
  const GatedAct ga{act, limit};
  if (I <= 0 || K <= 0 || w_rows != 2 * f8_padded_rows(I) || !act_known(ga) || ((uintptr_t)codes & 15)) return SHARPI_ERR_ARG;
  const F8Tiles p{(const uint8_t*)x, (const uint8_t*)x_scales, (const uint8_t*)w_codes, (const uint8_t*)w_scales, f8_blocks(K), w_rows, a_rows, offsets, rows, groups, (uint32_t)((long long)x_rows * f8_blocks(K) * kF8Block), along, height, 0, 0, 1};
  if (!tiles_ok(p, x_rows)) return SHARPI_ERR_ARG;
  return launch_tiles<true>(p, F8Out{nullptr, (uint8_t*)codes, (uint8_t*)scales, score, I}, ga, 2, DT_BF16, stream);
}
