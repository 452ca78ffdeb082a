// Softmax cross entropy of an output head, and its gradient, without keeping
// the logits.
//
//   s = h w^T            h [m, k], w [v, k] (rows of the vocabulary), bf16 or f16
//   lse_i = log sum_j exp(s_ij)         loss_i = lse_i - s_{i,t_i}
//   d_ij = g_i (exp(s_ij - lse_i) - [j = t_i])      dh = d w      dw = d^T h
//
// w is taken in the embedding's order [v, k]: its rows start on 16-byte
// boundaries for any v, so an odd vocabulary needs no padded copy.
//
// All three products run on one persistent CTA-pair tcgen05 mainloop (256 x 256
// tiles, cta_group::2, the roles of gemm_tcgen05_pair) with three epilogues:
//
//   kLse      tiles of s stay in tensor memory; each thread owns a row and keeps
//             a running maximum and sum of exponentials over the tile's words
//             other than the target. (max, sum) per row and tile go to the
//             workspace, and ce_stats joins them: with r the log-sum-exp over
//             the other words, loss = log(1 + exp(r - s_t)) keeps its digits
//             when the target is almost certain, where lse - s_t would cancel.
//             s_t itself, often the largest logit by far and so the one that
//             the tensor core's truncating accumulation moves most (4e-5 at
//             k = 4096), is a dot product of its own in fp32 lanes. The other
//             words' logits are taken as they are, a sum over k that is cut off
//             and not rounded at each step: at k = 4096 a row's loss is 9e-7 off,
//             where a plain fp32 product leaves 7e-7, but all to one side, so the
//             mean over rows is 1e-6 off (3e-7). Sums over k in two or four parts,
//             held in registers between them, halved and quartered that and took
//             2.5% and 4.7% more time (2048 rows; 10% and 12% with 256): not taken.
//             Up to 64 rows (ce_narrow) such parts cost nothing, and are.
//   kDlogits  a piece of the vocabulary at a time, s is formed again and leaves as
//             d, rounded to the operand type, in the workspace [rows, piece].
//             The target's entry is g (p_t - 1) = g expm1(-loss).
//   kGrads    both products of d for that piece in one launch: tiles of dh (d as
//             it lies, contracted over the piece, added to an fp32 accumulator
//             until the last piece) and tiles of dw (d transposed, taken by TMA as
//             an MN-major A operand, contracted over the rows).
//
// Up to 128 rows, where memory is the bound, ce_narrow takes the place of the
// first two and ce_few of the third.
//
// The gradient works on the rows that count: ce_grad_rows moves them to the
// front (a copy of h, a few microseconds) and hands the later kernels their
// number on the device, so ignored rows cost nothing and whatever they hold
// (NaN, infinities) reaches nothing.
//
// d is held with g scaled so that the largest |g| is 1 (f16: 2^14), and the
// epilogues of the products undo it in fp32. So the rounding of d is that of p and
// p_t - 1, not one that a common g (1 / rows, for the mean) would give every row
// alike, off by up to half a step of the type in one direction; and in f16
// probabilities down to 2^-28 keep their digits (in a row of the largest weight: an
// entry of d is off by up to 2^-39 of that). 16 bits, because the tensor core
// multiplies d with 16-bit w and h: two terms a value would cost the products a
// second time. Against 64 bits dh and dw are 0.0019 off (bf16; 0.00025 in f16), where
// rounding exact results alone is 0.0017 (0.00021).
#include <type_traits>

#include "tcgen05.cuh"

namespace axon {

__device__ int g_ce_error;

namespace {

constexpr int BM = 128;              // rows per CTA; 256 per pair
constexpr int BN = 256;              // columns per pair
constexpr int BH = BN / 2;           // columns staged per CTA
constexpr int BK = 64;               // 16-bit elements per 128-byte swizzle row
constexpr int A_BYTES = BM * BK * 2;
constexpr int B_BYTES = BH * BK * 2;
constexpr int STAGE = A_BYTES + B_BYTES;
constexpr int CHUNK = 64 * BK * 2;   // one 64 x 64 block of an MN-major operand
constexpr int kStaging = 32 * 128;   // 32 rows x 128 bytes for each warp that writes tiles
constexpr uint32_t TMEM_COLS = 2 * BN;
constexpr float kLog2e = 1.4426950408889634f;

enum Mode { kLse = 0, kDlogits = 1, kGrads = 2 };

// Epilogue warps: two share a TMEM lane quarter, half the columns each. Stages:
// as many of 32 KB as fit the 227 KB.
constexpr int kEpiWarps = 8;
constexpr int kPairThreads = 64 + 32 * kEpiWarps;
constexpr int stages_of(int mode) { return mode == kLse ? 7 : 6; }
constexpr int staging_of(int mode) { return mode == kLse ? 0 : kEpiWarps * kStaging; }
constexpr int smem_of(int mode) { return stages_of(mode) * STAGE + staging_of(mode) + 1024 + 256; }

// What ce_grad_rows hands to the kernels after it.
struct RowHeader {
  int rows;         // rows that count
  float unscale;    // what d must be multiplied by (see products_scale)
};

struct CeParams {
  CUtensorMap a, b;     // kLse, kDlogits: h, w.   kGrads and ce_few, dh tiles: d, w's piece
  CUtensorMap a2, b2;   // kGrads, dw tiles: d transposed, h
  CUtensorMap c;        // what the epilogue writes by TMA: kDlogits d, kGrads dw
  int m, v, k;          // rows (at most), words of this piece, hidden size
  const RowHeader* header;  // NULL: all m rows
  // kLse
  const void* targets;
  int target64;
  int64_t ignore_index;
  float2* part;         // [m][parts]
  int parts;            // half word tiles (ce_pair) or CTAs (ce_narrow)
  unsigned* done;       // counts ce_stats' CTAs; set to 0 here
  // kDlogits: per counted row
  const int* row_target;
  const float* row_lse;
  const float* row_g;
  const float* row_dt;
  int v0;               // first word of the piece
  void* d;              // [m][ld_d]
  int64_t ld_d;
  // kGrads
  const int* row_index; // counted row -> row of dh
  void* dh;
  void* dw;
  int64_t ld_dh;
  float* acc;           // fp32 [splits][m][k]: dh between pieces, and its splits
  int first, last;      // this piece is the vocabulary's first / last
  int splits;           // parts that dh's contraction over the piece is cut into
  int few;              // ce_few's rows of a dh tile (32, 64 or 128), 0: ce_pair
  int word_tile;        // kLse, kDlogits: words a tile
  int band;             // row tiles of s visited together
};

// A target as a word index, -1 ignored, -2 out of range.
__device__ __forceinline__ int load_target(const void* p, int is64, int64_t i, int64_t ignore_index, int64_t v) {
  const int64_t t = is64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
  if (t == ignore_index) return -1;
  return t >= 0 && t < v ? static_cast<int>(t) : -2;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp(x - ref): one ex2.approx, off by 2^-22 of itself and, from its argument's
// rounding, by 2^-24 of |x - ref|. expf would take several instructions more for
// each of m x v logits, whose own error is larger.
__device__ __forceinline__ float exp_from(float x, float ref) { return ex2((x - ref) * kLog2e); }

// mbar_wait by a whole warp, with one answer for all its lanes: where a wait
// gives up, no lane goes on to the warp-wide instructions behind it alone.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, &g_ce_error));
}

// Whether a wait gave up before this kernel (and nobody has asked for the status
// since): what the workspace holds is then not to be trusted, and the kernels
// that form the results write NaN. Asked once a thread, after pdl_wait.
__device__ __forceinline__ bool gave_up() { return *static_cast<volatile int*>(&g_ce_error) != 0; }

// ---- tiles -----------------------------------------------------------------------------

struct Tile {
  bool dw;          // kGrads: a tile of dw (else of dh)
  int tm, tn;       // row tile, column tile
  int k0, kb;       // first k-block, k-blocks
  int split;        // kGrads, dh: which part of the contraction
};

// What a tile costs beside its k-blocks, in k-blocks: filling the pipeline and
// writing 128 KB.
constexpr int kTileCost = 4;

// Up to this many k-blocks a dw tile takes longer to write than to compute.
constexpr int kFewRows = 8;

// A pair's way through the tiles, worked out once.
//
// kLse, kDlogits: bands of `band` row tiles (so that a band of h stays in L2),
// each band word tile by word tile.
//
// kGrads: the dh tiles (a contraction over the whole piece, or one part of it)
// are dealt in turn; the pairs that got one fewer take as many dw tiles as fit in
// one dh tile's time, and the rest of the dw tiles is dealt in turn. Row tiles run
// fastest for dh and column tiles for dw, so that the pairs share the words,
// and d, in L2. With few rows, even pairs begin with dh and odd ones with dw: dh is
// then bound by reading w and dw by writing, and memory that only writes moves
// 3.9 TB/s here, against 6.6 both ways (6% off the gradients of 64 x 2048 x 32000
// when they ran here; with 4096 rows it would cost 4%).
template <int MODE>
struct Walk {
  int pair, pairs, rows;
  int row_tiles, word_tiles, col_tiles;
  int kb_all, kb_dh, kb_dw;
  int mine, mine_dw, early, odd, behind;

  __device__ __forceinline__ Walk(const CeParams& p, int rows_) {
    pair = blockIdx.x >> 1;
    pairs = gridDim.x >> 1;
    rows = rows_;
    row_tiles = (rows + 2 * BM - 1) / (2 * BM);
    if constexpr (MODE != kGrads) {
      word_tiles = (p.v + p.word_tile - 1) / p.word_tile;
      kb_all = (p.k + BK - 1) / BK;
    } else {
      word_tiles = (p.v + 2 * BM - 1) / (2 * BM);
      col_tiles = (p.k + BN - 1) / BN;
      const int n_dh = p.dh ? row_tiles * col_tiles * p.splits : 0;
      const int n_dw = p.dw ? word_tiles * col_tiles : 0;
      kb_all = (p.v + BK - 1) / BK;
      kb_dh = (kb_all + p.splits - 1) / p.splits;
      kb_dw = (rows + BK - 1) / BK;
      odd = n_dh % pairs;  // pairs below this one have a dh tile more
      mine = n_dh / pairs + (pair < odd ? 1 : 0);
      behind = odd ? pairs - odd : 0;                      // pairs with one dh tile fewer
      early = (kb_dh + kTileCost) / (kb_dw + kTileCost);   // dw tiles they take meanwhile
      if (behind == 0) early = 0;
      else if (early > n_dw / behind) early = n_dw / behind;
      const int rest = n_dw - behind * early;
      mine_dw = (rest > pair ? (rest - pair + pairs - 1) / pairs : 0) + (pair >= odd ? early : 0);
    }
  }

  // The `i`-th tile of this pair; false past the last one.
  __device__ __forceinline__ bool at(const CeParams& p, int i, Tile& t) const {
    t.dw = false;
    t.k0 = 0;
    t.split = 0;
    if constexpr (MODE != kGrads) {
      int64_t at = static_cast<int64_t>(i) * pairs + pair;
      if (at >= static_cast<int64_t>(row_tiles) * word_tiles) return false;
      int first = 0, tiles = row_tiles;
      if (row_tiles > p.band) {
        const int64_t per_band = static_cast<int64_t>(p.band) * word_tiles;
        first = static_cast<int>(at / per_band) * p.band;
        at -= static_cast<int64_t>(first) * word_tiles;
        tiles = row_tiles - first < p.band ? row_tiles - first : p.band;
      }
      t.tn = static_cast<int>(at / tiles);
      t.tm = first + static_cast<int>(at - static_cast<int64_t>(t.tn) * tiles);
      t.kb = kb_all;
      return true;
    } else {
      if (i >= mine + mine_dw) return false;
      if ((pair & 1) && kb_dw <= kFewRows) i = i < mine_dw ? mine + i : i - mine_dw;
      if (i < mine) {
        const int at = i * pairs + pair, rest = at / row_tiles;
        t.tm = at - rest * row_tiles;
        t.split = rest / col_tiles;
        t.tn = rest - t.split * col_tiles;
        t.k0 = t.split * kb_dh;
        const int left = kb_all - t.k0;
        t.kb = left < kb_dh ? (left > 0 ? left : 0) : kb_dh;
        return true;
      }
      i -= mine;
      t.dw = true;
      t.kb = kb_dw;
      int at;
      if (pair >= odd && i < early) at = i * behind + (pair - odd);
      else at = behind * early + (i - (pair >= odd ? early : 0)) * pairs + pair;
      t.tm = at / col_tiles;
      t.tn = at - t.tm * col_tiles;
      return true;
    }
  }
};

// One k-block of this CTA's half of the operands: 128 rows of A, 128 columns
// of B, 32 KB. K-major operands come as 128 rows x 64 elements of k; MN-major
// ones as two blocks of 64 elements x 64 rows of k.
template <int MODE>
__device__ __forceinline__ void load_stage(const CeParams& p, const Tile& t, int kb, int rank, uint8_t* sa,
                                           uint32_t full) {
  kb += t.k0;
  uint8_t* sb = sa + A_BYTES;
  const int row0 = t.tm * 2 * BM + rank * BM;
  if constexpr (MODE != kGrads) {
    tma_load_2d_pair(&p.a, full, sa, kb * BK, row0);
    tma_load_2d_pair(&p.b, full, sb, kb * BK, t.tn * p.word_tile + rank * (p.word_tile / 2));
  } else {
    const int col0 = t.tn * BN + rank * BH;
    if (!t.dw) {
      tma_load_2d_pair(&p.a, full, sa, kb * BK, row0);
    } else {
      tma_load_2d_pair(&p.a2, full, sa, row0, kb * BK);
      tma_load_2d_pair(&p.a2, full, sa + CHUNK, row0 + 64, kb * BK);
    }
    const CUtensorMap* mb = t.dw ? &p.b2 : &p.b;
    tma_load_2d_pair(mb, full, sb, col0, kb * BK);
    tma_load_2d_pair(mb, full, sb + CHUNK, col0 + 64, kb * BK);
  }
}

// tcgen05 instruction descriptor: fp32 accumulator, M rows (256 a pair), N columns; bit 15 / 16:
// A / B is MN-major.
template <typename T>
__device__ __forceinline__ uint32_t idesc(int n, bool a_mn, bool b_mn, int m = 2 * BM) {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// ---- epilogues -----------------------------------------------------------------------

// What the products of d are multiplied by.
__device__ __forceinline__ float products_scale(const RowHeader* header) {
  return gave_up() ? __int_as_float(0x7fc00000) : header->unscale;
}

// Waits for this thread's TMEM loads, and ties the 32 registers of one of them to
// the wait, so that nothing reads them before it.
__device__ __forceinline__ void tmem_wait_ld32(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                 "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}

// tmem_wait_ld32 for 16 registers.
__device__ __forceinline__ void tmem_wait_ld16(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}

// COLS accumulator columns from tensor memory.
template <int COLS>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, float* v) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < COLS; i += 32) tmem_ld32(taddr + i, v + i);
#pragma unroll
  for (int i = 0; i < COLS; i += 32) tmem_wait_ld32(v + i);
}

__device__ __forceinline__ float max32(const float* v) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = fmaxf(fmaxf(v[i], v[i + 8]), fmaxf(v[i + 16], v[i + 24]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) a[i] = fmaxf(a[i], a[i + o]);
  return a[0];
}

// This warp is done with the accumulator (its values are in registers).
__device__ __forceinline__ void release_tmem(uint32_t leader_tempty, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive_cluster(leader_tempty, 1);
}

// 32 more words into a row's running maximum and sum; `left` of them count, and
// the one at `target` (negative or past 31: none) does not.
__device__ __forceinline__ void lse_words(float* v, int left, int target, float& mx, float& sum) {
  const float ninf = __int_as_float(0xff800000);
  if (left < 32) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j >= left) v[j] = ninf;
  }
  if (target >= 0 && target < 32) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (target == j) v[j] = ninf;
  }
  const float nm = fmaxf(mx, max32(v));
  const float ref = nm == ninf ? 0.f : nm;  // nothing counted yet: exp gives 0
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 32; ++j) s[j & 3] += exp_from(v[j], ref);
  sum = sum * exp_from(mx, ref) + ((s[0] + s[1]) + (s[2] + s[3]));
  mx = nm;
}

// kLse: this thread's row over half of the tile's words, the next 32 on their way
// from tensor memory (a load takes some 450 cycles) while 32 are worked on.
__device__ __forceinline__ void lse_tile(const CeParams& p, const Tile& t, uint32_t tbase, int half, int64_t row,
                                         bool row_ok, int target, int lane, uint32_t tempty) {
  const int words = p.word_tile / 2, at = half * words, col = t.tn * p.word_tile + at;
  const int count = min(words, p.v - col);  // the same for the whole warp; may be negative
  target -= col;
  float mx = __int_as_float(0xff800000), sum = 0.f;
  float a[32], b[32];
  __syncwarp();
  if (count > 0) tmem_ld32(tbase + at, a);
#pragma unroll 1
  for (int c = 0; c < count; c += 64) {
    tmem_wait_ld32(a);
    if (c + 32 < count) tmem_ld32(tbase + at + c + 32, b);
    lse_words(a, count - c, target - c, mx, sum);
    if (c + 32 >= count) break;
    tmem_wait_ld32(b);
    if (c + 64 < count) tmem_ld32(tbase + at + c + 64, a);
    lse_words(b, count - c - 32, target - c - 32, mx, sum);
  }
  release_tmem(tempty, lane);
  if (row_ok) p.part[row * p.parts + t.tn * 2 + half] = make_float2(mx, sum);
}

// A thread holds a row of an accumulator tile, so its stores would touch 32 rows
// an instruction. A warp's 32 rows x 128 bytes turn around in shared memory
// instead, 16-byte pieces in the order of TMA's 128-byte swizzle, and leave by a
// TMA store or in whole 128-byte row pieces.
__device__ __forceinline__ uint4* staged(uint8_t* stg, int row, int piece) {
  return reinterpret_cast<uint4*>(stg + row * 128 + ((piece ^ (row & 7)) << 4));
}

// This thread's row piece of 128 bytes into the staging memory.
template <typename T>
__device__ __forceinline__ void stage_row(uint8_t* stg, int lane, const float* v) {
  constexpr int E = Vec<T>::E;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    Vec<T> pk;
#pragma unroll
    for (int e = 0; e < E; ++e) pk.e[e] = from_f<T>(v[i * E + e]);
    *staged(stg, lane, i) = pk.u;
  }
}

// The staged rows to (col, row) of the map, once all lanes have written theirs.
__device__ __forceinline__ void store_staged(const CUtensorMap* map, uint8_t* stg, int lane, int col, int row) {
  fence_async_smem();
  __syncwarp();
  if (lane == 0) tma_store_2d(map, stg, col, row);
}

// Before the staging memory is written again: all but the last LEFT stores have
// read theirs.
template <int LEFT = 0>
__device__ __forceinline__ void staging_free(int lane) {
  if (lane == 0) tma_store_wait_read<LEFT>();
  __syncwarp();
}

// Rows of d that the contraction over rows reads: the counted ones up to the
// end of their k-block. Those past the counted ones are written as zeros; past
// m TMA reads zeros by itself.
__device__ __forceinline__ int rows_read(const CeParams& p, int rows) {
  const int end = (rows + BK - 1) / BK * BK;
  return end < p.m ? end : p.m;
}

// kDlogits: d for this thread's row in one half of the tile's words, 64 at a
// time; where that does not divide, the last 64 begin earlier and write some
// words a second time. The accumulator is released once the last are in
// registers.
template <typename T>
__device__ __forceinline__ void dlogits_tile(const CeParams& p, const Tile& t, uint32_t tbase, int half, int64_t row0,
                                             int lane, int rows, uint8_t* stg, uint32_t tempty) {
  const int64_t row = row0 + lane;
  const bool row_ok = row < rows, any = row0 < rows_read(p, rows);
  const float lse = row_ok ? p.row_lse[row] : 0.f;
  const float g = row_ok ? p.row_g[row] : 0.f;
  const float dt = row_ok ? p.row_dt[row] : 0.f;
  const int target = row_ok ? p.row_target[row] - p.v0 : -1;
#pragma unroll 1
  for (int c = 0, words = p.word_tile / 2; c < words; c += 64) {
    const int at = half * words + (c + 64 > words ? words - 64 : c), col = t.tn * p.word_tile + at;
    float v[64];
    tmem_ld_cols<64>(tbase + at, v);
    if (c + 64 >= words) release_tmem(tempty, lane);
    if (!any || col >= p.v) continue;  // the same for the whole warp
    const int left = row_ok ? p.v - col : 0;  // words of this piece that count
#pragma unroll
    for (int j = 0; j < 64; ++j) v[j] = j < left ? exp_from(v[j], lse) * g : 0.f;
    if (target >= col && target < col + 64) {
#pragma unroll
      for (int j = 0; j < 64; ++j)
        if (target == col + j) v[j] = dt;
    }
    staging_free(lane);
    stage_row<T>(stg, lane, v);
    store_staged(&p.c, stg, lane, col, static_cast<int>(row0));
  }
}

// Eight outputs rounded to TO (16-bit: one packet; fp32: two).
template <typename TO>
__device__ __forceinline__ void store8(TO* dst, const float* v) {
  if constexpr (sizeof(TO) == 4) {
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    Vec<TO> pk;
#pragma unroll
    for (int e = 0; e < 8; ++e) pk.e[e] = from_f<TO>(v[e]);
    st_vec(dst, pk);
  }
}

// Columns [c0, c0 + 128) of a tile of dw, rounded (row0 the warp's first
// word within the piece). The accumulator is released once its last part is in
// registers: with few rows a tile is one or two k-blocks, and its MMA would wait
// for the epilogue. BUFS staging buffers are used in turn.
template <typename TW, int BUFS>
__device__ __forceinline__ void dw_tile(const CeParams& p, int tn, int kb, uint32_t tbase, int c0, int64_t row0,
                                        int lane, float unscale, uint8_t* staging, uint32_t& turn, uint32_t tempty) {
  constexpr int COLS = 128 / sizeof(TW);
#pragma unroll 1
  for (int c = 0; c < BN / 2; c += COLS) {
    const int col = tn * BN + c0 + c;
    float v[COLS];
    tmem_ld_cols<COLS>(tbase + c0 + c, v);
    if (c + COLS == BN / 2) release_tmem(tempty, lane);
    if (row0 >= p.v || col >= p.k) continue;  // the same for the whole warp
#pragma unroll
    for (int j = 0; j < COLS; ++j) v[j] = kb ? v[j] * unscale : 0.f;  // no k-block: nothing was accumulated
    uint8_t* stg = staging + turn * kStaging;
    staging_free<BUFS - 1>(lane);
    stage_row<TW>(stg, lane, v);
    store_staged(&p.c, stg, lane, col, static_cast<int>(row0));
    if (BUFS > 1) turn ^= 1u;
  }
}

// kGrads, columns [c0, c0 + 128) of a tile of dh: added to the accumulator of its
// split, or, where this piece and part are all there is left, rounded and
// written to its row.
template <typename T>
__device__ __forceinline__ void dh_tile(const CeParams& p, const Tile& t, uint32_t tbase, int c0, int64_t row0,
                                        int lane, int rows, float unscale, uint8_t* stg, uint32_t tempty) {
  const bool direct = p.last && p.splits == 1;
  float* acc = p.acc + (static_cast<int64_t>(t.split) * p.m + row0) * p.k;
  staging_free(lane);
#pragma unroll 1
  for (int c = c0; c < c0 + BN / 2; c += 32) {
    const int col = t.tn * BN + c;
    if (col >= p.k) break;
    float v[32];
    tmem_ld_cols<32>(tbase + c, v);
    if (t.kb == 0) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = 0.f;
    }
    stage_row<float>(stg, lane, v);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + (lane >> 3), piece = lane & 7;
      if (row0 + r < rows && col + piece * 4 < p.k) {
        float4 x = *reinterpret_cast<const float4*>(staged(stg, r, piece));
        float4* at = reinterpret_cast<float4*>(acc + static_cast<int64_t>(r) * p.k + col + piece * 4);
        if (!p.first) {
          const float4 a = *at;
          x.x += a.x; x.y += a.y; x.z += a.z; x.w += a.w;
        }
        if (direct) {
          T* out = static_cast<T*>(p.dh) + p.row_index[row0 + r] * p.ld_dh + col + piece * 4;
          union { T e[4]; uint2 u; } pk;
          pk.e[0] = from_f<T>(x.x * unscale); pk.e[1] = from_f<T>(x.y * unscale);
          pk.e[2] = from_f<T>(x.z * unscale); pk.e[3] = from_f<T>(x.w * unscale);
          *reinterpret_cast<uint2*>(out) = pk.u;
        } else {
          *at = x;
        }
      }
    }
    __syncwarp();
  }
  release_tmem(tempty, lane);
}

// ---- the CTA-pair kernel ---------------------------------------------------------------
//
// Bound by the tensor pipe from some 300 rows up: it is 85-87% active in the three
// modes at 2048 x 4096 x 65536, where the loss runs 1549 TFLOP/s, d 1521 and the
// products 1494 in a burst (cuBLAS here: 1583). At hidden sizes of 512 and less the
// epilogue shows: 3.1 us a tile at k = 64 (reading 128 KB of tensor memory, the
// exponentials, and the tile's latencies), against 2.2 us of MMA at k = 512.

template <int MODE, typename T, typename TW>
__global__ void __launch_bounds__(kPairThreads, 1) ce_pair(const __grid_constant__ CeParams p) {
  constexpr int kStages = stages_of(MODE);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + kStages * STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + staging_of(MODE));
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* issued = reinterpret_cast<int*>(tmem_slot + 2);

  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const bool leader = rank == 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * kEpiWarps);  // one arrival per epilogue warp of each CTA
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *issued = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  cluster_barrier();  // both CTAs' barriers are initialised before either is addressed remotely
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  const Walk<MODE> w(p, p.header ? p.header->rows : p.m);
  Tile t;

  if (MODE == kLse && blockIdx.x == 0 && threadIdx.x == 64) *p.done = 0;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    const uint32_t pair_bytes = MODE == kGrads ? 2 * STAGE : 2 * A_BYTES + p.word_tile * BK * 2;
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; w.at(p, i, t); ++i) {
      for (int kb = 0; kb < t.kb; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, &g_ce_error)) goto producer_done;
        const uint32_t leader_full = mapa_u32(smem_u32(&full[stage]), 0);
        if (leader) mbar_expect_tx(&full[stage], pair_bytes);
        load_stage<MODE>(p, t, kb, static_cast<int>(rank), smem + stage * STAGE, leader_full);
        *issued += 1;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  producer_done:;
  } else if (warp == 1 && lane == 0 && leader) {
    // ---------------- MMA issuer (leader only) ----------------
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; w.at(p, i, t); ++i) {
      const int buf = i & 1;
      if (!mbar_wait(&tempty[buf], ((i >> 1) & 1) ^ 1u, abort_flag, &g_ce_error)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + static_cast<uint32_t>(buf * BN);
      const bool a_mn = MODE == kGrads && t.dw, b_mn = MODE == kGrads;
      const uint32_t id = idesc<T>(MODE == kGrads ? BN : p.word_tile, a_mn, b_mn);
      // one K = 16 step: 32 bytes along a K-major row, 16 rows of an MN-major block
      const uint32_t a_step = a_mn ? 2048 : 32, a_lbo = a_mn ? CHUNK : 16;
      const uint32_t b_step = b_mn ? 2048 : 32, b_lbo = b_mn ? CHUNK : 16;
      bool ok = true;
      for (int kb = 0; kb < t.kb; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, &g_ce_error)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * STAGE);
        const uint32_t sb = sa + A_BYTES;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          tc_mma_pair(d, sdesc(sa + k * a_step, a_lbo, 1024), sdesc(sb + k * b_step, b_lbo, 1024), id, (kb | k) != 0);
        tc_commit_to(smem_u32(&empty[stage]));
        tc_commit_to(mapa_u32(smem_u32(&empty[stage]), 1));
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      tc_commit_to(smem_u32(&tfull[buf]));
      tc_commit_to(mapa_u32(smem_u32(&tfull[buf]), 1));
    }
    // TMEM is released only after every MMA this thread issued has retired
    tc_commit_to(smem_u32(drain));
    volatile int never = 0;
    mbar_wait(drain, 0, &never, &g_ce_error);
  } else if (warp >= 2) {
    // ---------------- epilogue (both CTAs, their own 128 rows) ----------------
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    const float unscale = MODE == kGrads ? products_scale(p.header) : 1.f;
    uint32_t turn = 0;
    for (int i = 0; w.at(p, i, t); ++i) {
      const int buf = i & 1;
      const int64_t row0 = static_cast<int64_t>(t.tm) * 2 * BM + rank * BM + q * 32;  // of this warp's 32
      const bool row_ok = row0 + lane < w.rows;
      int target = -1;
      if (MODE == kLse && row_ok)  // on its way while the tile is computed
        target = load_target(p.targets, p.target64, row0 + lane, p.ignore_index, p.v);
      if (!warp_wait(&tfull[buf], (i >> 1) & 1, abort_flag)) break;
      tc_fence_after();
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(buf * BN);
      const uint32_t leader_tempty = mapa_u32(smem_u32(&tempty[buf]), 0);
      const int half = warp < 6 ? 0 : 1, c0 = half * (BN / 2);  // this warp's half of the columns
      if constexpr (MODE == kLse) {
        lse_tile(p, t, tbase, half, row0 + lane, row_ok, target, lane, leader_tempty);
      } else {
        uint8_t* stg = staging + (warp - 2) * kStaging;
        if constexpr (MODE == kDlogits) dlogits_tile<T>(p, t, tbase, half, row0, lane, w.rows, stg, leader_tempty);
        else if (t.dw) dw_tile<TW, 1>(p, t.tn, t.kb, tbase, c0, row0, lane, unscale, stg, turn, leader_tempty);
        else dh_tile<T>(p, t, tbase, c0, row0, lane, w.rows, unscale, stg, leader_tempty);
      }
    }
    if (MODE != kLse && lane == 0) tma_store_wait();
  }

  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag && *issued > 0) {
    // copies issued by this CTA may still be landing: give them time before
    // the pair leaves (this path only runs after a wait gave up)
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  cluster_barrier();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS)
                 : "memory");
  }
}

// ---- few rows: both products, read and written at once ---------------------------------------
//
// Up to 128 rows the products are bound by memory: dh reads w, dw is written.
// Memory that is only written moves 3.9 TB/s on this card and 6.6 both ways, so
// the two run at the same time on every SM, as two pipelines of one CTA that
// share nothing but the tensor pipe:
//
//   dh   transposed, 128 of its columns on the accumulator's lanes and the rows
//        beside them (A: w's words x columns as they lie, MN-major; B: d). A
//        k-block is 16 KB of w and 4-16 KB of d; two accumulators; warps 0
//        (TMA), 1 (MMA) and 12-15 (a warp's 32 lanes are 32 neighbouring
//        columns of a row).
//   dw   128 words x 256 columns, one or two k-blocks of rows, so all epilogue: one
//        accumulator, given back when its second half is in registers. A CTA
//        keeps to one block of columns, so its part of h stays in shared memory,
//        and neighbouring CTAs write neighbouring pieces of dw's rows. Warps 2
//        (TMA), 3 (MMA) and 4-11, TMA stores.
//
// Gradients in all: 64 rows x 2048 x 32000 94-97 us (one after the other on CTA
// pairs 105), one row x 4096 x 128256 591-598 us (620), where dw written alone takes
// 3.3 TB/s of the 3.9 and dh alone reads w at 6.4. Blocks of columns that do not
// divide the CTAs leave some without dw: 4 of 148 at k = 4096; above k = 18944 each
// block has one CTA, so 75 at the least write (not measured above 4096).
constexpr int kFewThreads = 512;
constexpr int kFewDwStages = 2;                                 // of d transposed, 16 KB
constexpr int few_h(int few) { return (few + BK - 1) / BK * 2 * B_BYTES; }  // h, 32 KB a k-block
constexpr int few_bufs(int few) { return few > 64 ? 1 : 2; }    // staging buffers a warp
constexpr int few_fixed(int few) {
  return kFewDwStages * A_BYTES + few_h(few) + 8 * few_bufs(few) * kStaging + 1024 + 256;
}
constexpr int few_stage(int few) { return A_BYTES + few * BK * 2; }
constexpr int few_stages(int few) { return (232448 - few_fixed(few)) / few_stage(few); }
constexpr int few_smem(int few) { return few_stages(few) * few_stage(few) + few_fixed(few); }

// 32 lanes x 16 consecutive 32-bit TMEM columns.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// A tile of dh, transposed: this thread's column (lane) of dh in every row.
template <typename T>
__device__ __forceinline__ void few_dh_tile(const CeParams& p, int split, int kb, uint32_t tbase, int64_t col, int lane,
                                            int rows, float unscale, uint32_t tempty) {
  const bool direct = p.last && p.splits == 1, ok = col < p.k;
  float* acc = p.acc + static_cast<int64_t>(split) * p.m * p.k + col;
#pragma unroll 1
  for (int r = 0; r < rows; r += 16) {
    float v[16];
    __syncwarp();
    tmem_ld16(tbase + r, v);
    tmem_wait_ld16(v);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (!ok || r + j >= rows) continue;
      float x = kb ? v[j] : 0.f;
      float* at = acc + static_cast<int64_t>(r + j) * p.k;
      if (!p.first) x += *at;
      if (direct) static_cast<T*>(p.dh)[p.row_index[r + j] * p.ld_dh + col] = from_f<T>(x * unscale);
      else *at = x;
    }
  }
  release_tmem(tempty, lane);
}

template <int FEW, typename T, typename TW>
__global__ void __launch_bounds__(kFewThreads, 1) ce_few(const __grid_constant__ CeParams p) {
  constexpr int S = few_stages(FEW), SB = few_stage(FEW), BUFS = few_bufs(FEW);
  static_assert(S >= 3, "w must be read ahead");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* dw_ring = smem + S * SB;
  uint8_t* h_block = dw_ring + kFewDwStages * A_BYTES;
  uint8_t* staging = h_block + few_h(FEW);
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + 8 * BUFS * kStaging);  // dh
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint64_t* dw_full = tempty + 2;
  uint64_t* dw_empty = dw_full + kFewDwStages;
  uint64_t* dw_tfull = dw_empty + kFewDwStages;
  uint64_t* dw_tempty = dw_tfull + 1;
  uint64_t* h_full = dw_tempty + 1;
  uint64_t* drain = h_full + 1;  // dh, dw
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* issued = reinterpret_cast<int*>(tmem_slot + 2);  // dh, dw

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 4);
      mbar_init(&drain[b], 1);
      issued[b] = 0;
    }
    for (int s = 0; s < kFewDwStages; ++s) {
      mbar_init(&dw_full[s], 1);
      mbar_init(&dw_empty[s], 1);
    }
    mbar_init(dw_tfull, 1);
    mbar_init(dw_tempty, 8);
    mbar_init(h_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  pdl_wait();
  pdl_trigger();
  const int rows = p.header->rows;
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t dw_tmem = tmem_base + BN;  // columns 256..511; dh's two accumulators are below

  // dh: columns run fastest, so that neighbouring CTAs read neighbouring pieces of w's rows
  const int dh_cols = (p.k + BM - 1) / BM;
  const int n_dh = p.dh && rows > 0 ? dh_cols * p.splits : 0;
  const int kb_all = (p.v + BK - 1) / BK, kb_dh = (kb_all + p.splits - 1) / p.splits;
  const int dw_cols = (p.k + BN - 1) / BN;
  const int kb_dw = (rows + BK - 1) / BK;
  // dw: this CTA's block of columns, its first word tile and the step to the next
  const int tn = blockIdx.x % dw_cols, step = gridDim.x / dw_cols;
  const int tm0 = static_cast<int>(blockIdx.x) < step * dw_cols ? blockIdx.x / dw_cols : INT32_MAX;
  const int word_tiles = p.dw ? (p.v + BM - 1) / BM : 0;

  if (warp == 0 && lane == 0) {
    // ---------------- dh: TMA ----------------
    int stage = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x; t < n_dh; t += gridDim.x) {
      const int split = t / dh_cols, col = (t - split * dh_cols) * BM;
      const int k1 = min(kb_all, (split + 1) * kb_dh);
      for (int kb = split * kb_dh; kb < k1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, &g_ce_error)) goto dh_loaded;
        mbar_expect_tx(&full[stage], static_cast<uint32_t>(SB));
        uint8_t* sa = smem + stage * SB;
        tma_load_2d(&p.b, &full[stage], sa, col, kb * BK);
        tma_load_2d(&p.b, &full[stage], sa + CHUNK, col + 64, kb * BK);
        tma_load_2d(&p.a, &full[stage], sa + A_BYTES, kb * BK, 0);
        issued[0] += 1;
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  dh_loaded:;
  } else if (warp == 1 && lane == 0) {
    // ---------------- dh: MMA ----------------
    const uint32_t id = idesc<T>(FEW, true, false, BM);
    int stage = 0, i = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x; t < n_dh; t += gridDim.x, ++i) {
      const int buf = i & 1;
      if (!mbar_wait(&tempty[buf], ((i >> 1) & 1) ^ 1u, abort_flag, &g_ce_error)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + static_cast<uint32_t>(buf * FEW);
      const int k0 = t / dh_cols * kb_dh, k1 = min(kb_all, k0 + kb_dh);
      bool ok = true;
      for (int kb = k0; kb < k1; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, &g_ce_error)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * SB);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          tc_mma(d, sdesc(sa + k * 2048, CHUNK, 1024), sdesc(sa + A_BYTES + k * 32, 16, 1024), id,
                 ((kb - k0) | k) != 0);
        tc_commit(&empty[stage]);
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      tc_commit(&tfull[buf]);
    }
    tc_commit(&drain[0]);  // TMEM is released only after every MMA has retired
    volatile int never = 0;
    mbar_wait(&drain[0], 0, &never, &g_ce_error);
  } else if (warp == 2 && lane == 0) {
    // ---------------- dw: TMA ----------------
    int stage = 0;
    uint32_t phase = 0;
    if (tm0 < word_tiles && kb_dw > 0) {
      mbar_expect_tx(h_full, static_cast<uint32_t>(kb_dw * 2 * B_BYTES));
      for (int i = 0; i < kb_dw * (BN / 64); ++i)
        tma_load_2d(&p.b2, h_full, h_block + i * CHUNK, tn * BN + i % (BN / 64) * 64, i / (BN / 64) * BK);
      issued[1] += 1;
    }
    for (int tm = tm0; tm < word_tiles; tm += step) {
      for (int kb = 0; kb < kb_dw; ++kb) {
        if (!mbar_wait(&dw_empty[stage], phase ^ 1u, abort_flag, &g_ce_error)) goto dw_loaded;
        mbar_expect_tx(&dw_full[stage], A_BYTES);
        uint8_t* sa = dw_ring + stage * A_BYTES;
        tma_load_2d(&p.a2, &dw_full[stage], sa, tm * BM, kb * BK);
        tma_load_2d(&p.a2, &dw_full[stage], sa + CHUNK, tm * BM + 64, kb * BK);
        if (++stage == kFewDwStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  dw_loaded:;
  } else if (warp == 3 && lane == 0) {
    // ---------------- dw: MMA ----------------
    const uint32_t id = idesc<T>(BN, true, true, BM);
    int stage = 0;
    uint32_t phase = 0, use = 0;
    for (int tm = tm0; tm < word_tiles; tm += step, use ^= 1u) {
      if (!mbar_wait(dw_tempty, use ^ 1u, abort_flag, &g_ce_error)) break;
      bool ok = kb_dw == 0 || tm != tm0 || mbar_wait(h_full, 0, abort_flag, &g_ce_error);
      if (!ok) break;
      tc_fence_after();
      for (int kb = 0; kb < kb_dw; ++kb) {
        if (!mbar_wait(&dw_full[stage], phase, abort_flag, &g_ce_error)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sa = smem_u32(dw_ring + stage * A_BYTES), sb = smem_u32(h_block + kb * 2 * B_BYTES);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          tc_mma(dw_tmem, sdesc(sa + k * 2048, CHUNK, 1024), sdesc(sb + k * 2048, CHUNK, 1024), id, (kb | k) != 0);
        tc_commit(&dw_empty[stage]);
        if (++stage == kFewDwStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      tc_commit(dw_tfull);
    }
    tc_commit(&drain[1]);
    volatile int never = 0;
    mbar_wait(&drain[1], 0, &never, &g_ce_error);
  } else if (warp >= 12) {
    // ---------------- dh: epilogue ----------------
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    const float unscale = products_scale(p.header);
    int i = 0;
    for (int t = blockIdx.x; t < n_dh; t += gridDim.x, ++i) {
      const int buf = i & 1;
      if (!warp_wait(&tfull[buf], (i >> 1) & 1, abort_flag)) break;
      tc_fence_after();
      const int split = t / dh_cols, kb = min(kb_all, (split + 1) * kb_dh) - split * kb_dh;
      const int64_t col = static_cast<int64_t>(t - split * dh_cols) * BM + q * 32 + lane;
      few_dh_tile<T>(p, split, kb > 0 ? kb : 0, tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * FEW, col,
                     lane, rows, unscale, mapa_u32(smem_u32(&tempty[buf]), 0));
    }
  } else if (warp >= 4) {
    // ---------------- dw: epilogue ----------------
    const int q = warp & 3, c0 = warp < 8 ? 0 : BN / 2;
    const float unscale = products_scale(p.header);
    uint8_t* stg = staging + (warp - 4) * BUFS * kStaging;
    uint32_t use = 0, turn = 0;
    for (int tm = tm0; tm < word_tiles; tm += step, use ^= 1u) {
      if (!warp_wait(dw_tfull, use, abort_flag)) break;
      tc_fence_after();
      dw_tile<TW, BUFS>(p, tn, kb_dw, dw_tmem + (static_cast<uint32_t>(q * 32) << 16), c0,
                        static_cast<int64_t>(tm) * BM + q * 32, lane, unscale, stg, turn,
                        mapa_u32(smem_u32(dw_tempty), 0));
    }
    if (lane == 0) tma_store_wait();
  }

  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag && (issued[0] > 0 || issued[1] > 0)) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // copies issued may still be landing
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// ---- few rows: the words on the accumulator's lanes -----------------------------------------
//
// With at most 128 rows the products are bound by reading w once, and a tile of
// 256 rows by 256 words would spend its shared memory and MMA time on rows that
// are not there. Here the words are the MMA's M (up to 128 a tile, one CTA) and
// the rows its N (NT = 16 to 128), so a k-block stages 16 KB of w beside 2-16 KB
// of h, six to twelve of them deep. The words a tile holds are chosen so that
// all CTAs get the same number of tiles.
//
//   kLse      a thread owns a lane, so one word of each of its CTA's tiles, and
//             keeps a running (max, sum) for every row in registers; the 128
//             lanes are joined once, at the end, into one (max, sum) per row
//             and CTA;
//   kDlogits  a warp's 32 lanes are 32 neighbouring words of a row of d.
//
// One row against 128256 words of 4096: 170 us as called, ce_stats and all, 6.2 TB/s
// (0.95 of a copy's rate; the 256-row tiles took 256). 64 rows x 2048 x 32000: 31 us,
// 4.2 TB/s. 128 rows x 4096 x 128256: 193 us in a burst (212), 223 at a clock that the
// power cap holds down.
constexpr int kNarrowRows = 128;
constexpr int kNarrowMaxStages = 12;

constexpr int narrow_stage(int nt) { return A_BYTES + nt * BK * 2; }
// Per row: the target (kLse), or what its entries of d need (kDlogits).
constexpr int narrow_row_bytes(int mode) { return mode == kLse ? 4 : 16; }
constexpr int narrow_extra(int mode, int nt) { return 1024 + 256 + nt * narrow_row_bytes(mode); }
constexpr int narrow_stages(int mode, int nt) {
  const int fit = (232448 - narrow_extra(mode, nt)) / narrow_stage(nt);
  return fit < kNarrowMaxStages ? fit : kNarrowMaxStages;
}
constexpr int narrow_smem(int mode, int nt) { return narrow_stages(mode, nt) * narrow_stage(nt) + narrow_extra(mode, nt); }
// Epilogue warps: each takes 32 of the rows (16 of 16) on its quarter of the lanes.
constexpr int narrow_cols(int nt) { return nt < 32 ? nt : 32; }
constexpr int narrow_epi_warps(int nt) { return 4 * nt / narrow_cols(nt); }
constexpr int narrow_threads(int nt) { return 64 + 32 * narrow_epi_warps(nt); }

// kLse: the parts that a sum over k is cut into at most, accumulators beside one
// another (512 columns for two tiles) that the epilogue adds in fp32. The tensor core
// cuts the sum off at each step and does not round it, always towards zero, so the
// error grows with the steps: in one part (256 steps at k = 4096) the loss of one row
// was 1.6e-6 off, in eight it is 1.9e-7 (sums in fp32 lanes: 2.7e-7), in the same
// time to 1% (reading w bounds it). With more than 64 rows there is room for two
// parts, which took 2.5% more time and halved 9.5e-7: not taken, as in ce_pair.
constexpr int narrow_parts(int mode, int nt) { return mode != kLse || nt > 64 ? 1 : nt > 32 ? 4 : 8; }
constexpr int kPartBlocks = 8;  // k-blocks of a part at least

// Joins (max, sum) pairs.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float mx = fmaxf(a.x, b.x);
  const float ref = mx == __int_as_float(0xff800000) ? 0.f : mx;
  return make_float2(mx, a.y * exp_from(a.x, ref) + b.y * exp_from(b.x, ref));
}

template <int MODE, typename T, int NT>
__global__ void __launch_bounds__(narrow_threads(NT), 1) ce_narrow(const __grid_constant__ CeParams p) {
  constexpr int S = narrow_stages(MODE, NT);
  constexpr int SB = narrow_stage(NT);
  constexpr int CW = narrow_cols(NT), EPI = 32 * narrow_epi_warps(NT);
  constexpr int PARTS = narrow_parts(MODE, NT);
  constexpr uint32_t COLS = 2 * NT * PARTS < 32 ? 32 : 2 * NT * PARTS;
  static_assert(S * SB >= 129 * NT * 8, "the lanes' pairs are joined in the stages' memory");
  static_assert((2 * S + 5) * 8 + 16 <= 256, "the rows' values begin 256 bytes behind the stages");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S * SB);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* issued = reinterpret_cast<int*>(tmem_slot + 2);
  int* row_target = reinterpret_cast<int*>(smem + S * SB + 256);       // kLse: [NT]
  float4* row_value = reinterpret_cast<float4*>(smem + S * SB + 256);  // kDlogits: [NT] lse, g, entry at the target, target

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], EPI / 32);  // one arrival per epilogue warp
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *issued = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  pdl_wait();
  pdl_trigger();
  const int rows = p.header ? p.header->rows : p.m;
  for (int r = threadIdx.x; r < NT; r += narrow_threads(NT)) {
    if constexpr (MODE == kLse)
      row_target[r] = r < rows ? load_target(p.targets, p.target64, r, p.ignore_index, p.v) : -1;
    else
      row_value[r] = r < rows ? make_float4(p.row_lse[r], p.row_g[r], p.row_dt[r],
                                            __int_as_float(p.row_target[r] - p.v0))
                              : make_float4(0.f, 0.f, 0.f, __int_as_float(-1));
  }
  if (MODE == kLse && blockIdx.x == 0 && threadIdx.x == 64) *p.done = 0;
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int tiles = rows > 0 ? (p.v + p.word_tile - 1) / p.word_tile : 0;
  const uint32_t stage_bytes = static_cast<uint32_t>(p.word_tile * BK * 2 + NT * BK * 2);
  const int kblocks = (p.k + BK - 1) / BK;
  const int part = PARTS > 1 ? max((kblocks + PARTS - 1) / PARTS, kPartBlocks) : kblocks;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer ----------------
    int stage = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x)
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, &g_ce_error)) goto producer_done;
        mbar_expect_tx(&full[stage], stage_bytes);
        uint8_t* sa = smem + stage * SB;
        tma_load_2d(&p.a, &full[stage], sa, kb * BK, t * p.word_tile);
        tma_load_2d(&p.b, &full[stage], sa + A_BYTES, kb * BK, 0);
        *issued += 1;
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
  producer_done:;
  } else if (warp == 1 && lane == 0) {
    // ---------------- MMA issuer ----------------
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t id = (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(NT >> 3) << 17) |
                            (static_cast<uint32_t>(BM >> 4) << 24);
    int stage = 0;
    uint32_t phase = 0;
    int i = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
      const int buf = i & 1;
      if (!mbar_wait(&tempty[buf], ((i >> 1) & 1) ^ 1u, abort_flag, &g_ce_error)) break;
      tc_fence_after();
      uint32_t d = tmem_base + static_cast<uint32_t>(buf * NT * PARTS);
      bool ok = true;
      for (int kb = 0, left = part; kb < kblocks; ++kb, --left) {
        if (!mbar_wait(&full[stage], phase, abort_flag, &g_ce_error)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (left == 0) {  // the next part
          d += NT;
          left = part;
        }
        const uint32_t sa = smem_u32(smem + stage * SB);
        const uint32_t sb = sa + A_BYTES;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          tc_mma(d, sdesc(sa + k * 32, 16, 1024), sdesc(sb + k * 32, 16, 1024), id, left != part || k != 0);
        tc_commit(&empty[stage]);
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      tc_commit(&tfull[buf]);
    }
    // TMEM is released only after every MMA this thread issued has retired
    tc_commit(drain);
    volatile int never = 0;
    mbar_wait(drain, 0, &never, &g_ce_error);
  } else if (warp >= 2) {
    // ---------------- epilogue ----------------
    const float ninf = __int_as_float(0xff800000);
    const int q = warp & 3;                 // TMEM lane quarter this warp may access
    const int c0 = (warp - 2) / 4 * CW;     // its first row
    float mx[MODE == kLse ? CW : 1], sm[MODE == kLse ? CW : 1];
    if constexpr (MODE == kLse) {
#pragma unroll
      for (int c = 0; c < CW; ++c) {
        mx[c] = ninf;
        sm[c] = 0.f;
      }
    }
    const int write = MODE == kDlogits ? rows_read(p, rows) : p.m;
    int i = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
      const int buf = i & 1;
      if (!warp_wait(&tfull[buf], (i >> 1) & 1, abort_flag)) break;
      tc_fence_after();
      // lanes past the tile's words hold what the stage held before
      const int word = q * 32 + lane < p.word_tile ? t * p.word_tile + q * 32 + lane : 0x7fffffff;
      const uint32_t tbase =
          tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(buf * NT * PARTS + c0);
      if (c0 < write) {  // the same for the whole warp
#pragma unroll
        for (int c1 = 0; c1 < CW; c1 += 16) {
          float v[16];
          __syncwarp();
          tmem_ld16(tbase + c1, v);
          tmem_wait_ld16(v);
          if constexpr (PARTS > 1) {
#pragma unroll 1
            for (int at = NT, kb = part; kb < kblocks; at += NT, kb += part) {
              float u[16];
              tmem_ld16(tbase + c1 + at, u);
              tmem_wait_ld16(u);
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] += u[j];
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int c = c1 + j;
            if constexpr (MODE == kLse) {
              const float x = word < p.v && row_target[c0 + c] != word ? v[j] : ninf;
              const float nm = fmaxf(mx[c], x);
              const float ref = nm == ninf ? 0.f : nm;
              sm[c] = sm[c] * exp_from(mx[c], ref) + exp_from(x, ref);
              mx[c] = nm;
            } else {
              const float4 r = row_value[c0 + c];
              float x = __float_as_int(r.w) == word ? r.z : exp_from(v[j], r.x) * r.y;
              if (word >= p.v || c0 + c >= rows) x = 0.f;
              if (c0 + c < write && word < p.ld_d) static_cast<T*>(p.d)[(c0 + c) * p.ld_d + word] = from_f<T>(x);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[buf]);
    }
    if constexpr (MODE == kLse) {
      // every stage has been read (the last accumulator is done): its memory
      // takes the lanes' pairs, 128 (and one of padding) for each row
      float2* lanes = reinterpret_cast<float2*>(smem);
      const int e = threadIdx.x - 64;
#pragma unroll
      for (int c = 0; c < CW; ++c) lanes[(c0 + c) * 129 + q * 32 + lane] = make_float2(mx[c], sm[c]);
      asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
      constexpr int SEG = EPI / NT, PER = 128 / SEG;  // threads that share a row, lanes each
      const float2* mine = lanes + (e % NT) * 129 + e / NT * PER;
      float2 s = make_float2(ninf, 0.f);
#pragma unroll 16
      for (int j = 0; j < PER; ++j) s.x = fmaxf(s.x, mine[j].x);
      const float ref = s.x == ninf ? 0.f : s.x;
#pragma unroll 16
      for (int j = 0; j < PER; ++j) s.y += mine[j].y * exp_from(mine[j].x, ref);
      asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
      lanes[e] = s;
      asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
      if (e < rows) {  // NT threads at most: rows <= NT
#pragma unroll
        for (int j = 1; j < SEG; ++j) s = join(s, lanes[j * NT + e]);
        p.part[static_cast<int64_t>(e) * p.parts + blockIdx.x] = s;
      }
    }
  }

  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag && *issued > 0) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // copies issued may still be landing
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLS) : "memory");
  }
}

// ---- the row kernels ---------------------------------------------------------------------

// Dot product of two rows of k 16-bit elements by one warp, in 8 x 32 fp32
// chains of k / 256 products each.
template <typename T>
__device__ __forceinline__ float warp_dot(const T* x, const T* y, int k, int lane) {
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = lane * 8; i < k; i += 256) {
    const Vec<T> a = ld_vec(x + i), b = ld_vec(y + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(to_f(a.e[e]), to_f(b.e[e]), acc[e]);
  }
  return warp_sum(((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7])));
}

// CTA-wide sums in a fixed order, returned to every thread.
template <typename V, int THREADS>
__device__ __forceinline__ V cta_sum(V v) {
  __shared__ V part[THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  V s = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) s += part[i];
  __syncthreads();
  return s;
}

struct StatsArgs {
  const void* h;
  const void* w;
  int64_t ld_h, ld_w;
  const float2* part;
  const void* targets;
  int target64;
  int64_t ignore_index;
  int m, k, v, parts;
  float* lse;
  float* loss_rows;
  float* loss_copy;   // the rows' losses a second time, or NULL
  float* loss;        // NULL: no sum or mean asked
  int mean;
  unsigned* done;
};

constexpr int kStatsThreads = 128;
constexpr int kStatsRows = kStatsThreads / 32;

// Joins a row's (max, sum) parts with the target's logit, a warp per row (27 us
// for 4096 rows of k = 4096, most of it the targets' rows of w); the
// CTA that comes last adds the rows' losses up, in row order whichever CTA it
// is, with its 128 threads: that sum grows with m alone (230 us for 131072 rows of
// k = 64, most of it this sum; a head of 4096 x 128256 takes some 90 ms for them).
template <typename T>
__global__ void __launch_bounds__(kStatsThreads) ce_stats(StatsArgs a) {
  const float ninf = __int_as_float(0xff800000);
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kStatsRows + (threadIdx.x >> 5);
  const int target = row < a.m ? load_target(a.targets, a.target64, row, a.ignore_index, a.v) : -1;
  float at = 0.f;
  if (target >= 0)  // reads only the caller's operands: need not wait for the kernel before
    at = warp_dot(static_cast<const T*>(a.h) + row * a.ld_h, static_cast<const T*>(a.w) + target * a.ld_w, a.k, lane);
  pdl_wait();
  if (row < a.m) {
    const float2* pr = a.part + row * a.parts;
    float mx = ninf;
    for (int i = lane; i < a.parts; i += 32) mx = fmaxf(mx, pr[i].x);
    mx = warp_max(mx);
    const float ref = mx == ninf ? 0.f : mx;
    float sum = 0.f;
    for (int i = lane; i < a.parts; i += 32) {
      const float2 t = pr[i];
      sum += t.y * exp_from(t.x, ref);
    }
    sum = warp_sum(sum);
    if (lane == 0) {
      const float log_sum = logf(sum);
      const float rest = ref + log_sum;  // the log-sum-exp over the words other than the target
      float lse = rest, loss = 0.f;
      if (target >= 0) {
        // loss = log(1 + y) with y the other words' odds against the target, so
        // that an almost certain target's loss keeps its digits. Past e^80 it is
        // log y: sum goes up to v, so y leaves fp32's range before exp(x) does.
        const float x = ref - at, log_y = x + log_sum;
        if (sum == 0.f) {  // no other word has a probability (v = 1, say)
          loss = at - at;  // 0, or NaN for an infinite logit
          lse = at;
        } else if (log_y > 80.f) {
          loss = log_y;
        } else {
          loss = log1pf(sum * expf(x));
          lse = at + loss;
        }
        if (at > 3.4e38f) loss = lse - at;  // an infinite logit: NaN, as lse - s_t says, not 0
      } else if (target == -2) {
        loss = __int_as_float(0x7fc00000);
      }
      if (gave_up()) lse = loss = __int_as_float(0x7fc00000);
      a.lse[row] = lse;
      a.loss_rows[row] = loss;
      if (a.loss_copy) a.loss_copy[row] = loss;
    }
  }
  if (!a.loss) return;
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(a.done, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  double sum = 0.0;
  int count = 0;
  for (int i = threadIdx.x; i < a.m; i += kStatsThreads) {
    sum += static_cast<double>(__ldcg(a.loss_rows + i));
    count += load_target(a.targets, a.target64, i, a.ignore_index, a.v) != -1;
  }
  sum = cta_sum<double, kStatsThreads>(sum);
  count = cta_sum<int, kStatsThreads>(count);
  if (threadIdx.x == 0) *a.loss = static_cast<float>(a.mean ? sum / static_cast<double>(count) : sum);
}

struct RowsArgs {
  const void* h;
  int64_t ld_h;
  const void* targets;
  int target64;
  int64_t ignore_index, v;
  const float* lse;
  const float* loss;
  const float* dloss;
  int per_row;        // dloss has a value per row (else one)
  int mean;
  int f16;
  int m, k;
  void* dh;           // rows that do not count become zero here; may be NULL
  int64_t ld_dh;
  RowHeader* header;
  int* row_index;
  int* row_target;
  float* row_lse;
  float* row_g;
  float* row_dt;
  void* hc;           // [m][k]
};

constexpr int kRowThreads = 256;

// Moves the rows that count to the front. Every CTA owns a range of rows; it
// finds the number of counted rows before its own, and the largest |g|, by
// reading all targets itself, where a second launch would cost more. Bound by the
// copy of h: 18 us at 4096 x 4096, 6 at 64 rows. The reads of the targets (and of
// dloss, one a row) grow with m times the CTAs, four an SM at most, from L2:
// 117 us in all for 131072 rows of k = 64, where d and its products take 845.
__global__ void __launch_bounds__(kRowThreads) ce_grad_rows(RowsArgs a) {
  __shared__ int slot[kRowThreads];
  __shared__ int warp_count[kRowThreads / 32];
  __shared__ float warp_top[kRowThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.m + gridDim.x - 1) / gridDim.x;
  const int r0 = min(a.m, static_cast<int>(blockIdx.x) * per), r1 = min(a.m, r0 + per);
  int before = 0, all = 0;
  float top = 0.f;
  pdl_wait();
  pdl_trigger();
  for (int i = tid; i < a.m; i += kRowThreads) {
    if (load_target(a.targets, a.target64, i, a.ignore_index, a.v) == -1) continue;
    all += 1;
    before += i < r0;
    top = fmaxf(top, fabsf(a.dloss[a.per_row ? i : 0]));
  }
  before = cta_sum<int, kRowThreads>(before);
  all = cta_sum<int, kRowThreads>(all);
  top = warp_max(top);
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
  for (int i = 0; i < kRowThreads / 32; ++i) top = fmaxf(top, warp_top[i]);
  const float unit = a.f16 ? 16384.f : 1.f;  // what the largest |g| becomes
  const bool scaled = top > 0.f && top < __int_as_float(0x7f800000);
  if (blockIdx.x == 0 && tid == 0) {
    const float weight = a.mean ? 1.f / static_cast<float>(all) : 1.f;
    *a.header = RowHeader{all, scaled ? top / unit * weight : weight};
  }

  const int packets = a.k / 8;
  for (int base = r0; base < r1; base += kRowThreads) {
    const int row = base + tid;
    int target = -1;
    if (row < r1) target = load_target(a.targets, a.target64, row, a.ignore_index, a.v);
    const bool counts = target != -1;
    const unsigned votes = __ballot_sync(0xffffffffu, counts);
    if (lane == 0) warp_count[warp] = __popc(votes);
    __syncthreads();
    int at = before + __popc(votes & ((1u << lane) - 1u));
    for (int i = 0; i < kRowThreads / 32; ++i) {
      if (i < warp) at += warp_count[i];
      before += warp_count[i];
    }
    slot[tid] = counts ? at : -1;
    if (counts) {
      float g = a.dloss[a.per_row ? row : 0];
      if (scaled) g = g / top * unit;
      if (target == -2) g = __int_as_float(0x7fc00000);  // a target outside the vocabulary poisons the gradients
      a.row_index[at] = row;
      a.row_target[at] = target;
      a.row_lse[at] = a.lse[row];
      a.row_g[at] = g;
      a.row_dt[at] = g * expm1f(-a.loss[row]);
    }
    __syncthreads();
    const int rows = min(kRowThreads, r1 - base);
    for (int64_t i = tid; i < static_cast<int64_t>(rows) * packets; i += kRowThreads) {
      const int r = static_cast<int>(i / packets);
      const int c = static_cast<int>(i - static_cast<int64_t>(r) * packets);
      const int to = slot[r];
      if (to >= 0) {
        static_cast<uint4*>(a.hc)[static_cast<int64_t>(to) * packets + c] =
            reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.h) + (base + r) * a.ld_h)[c];
      } else if (a.dh) {
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dh) + (base + r) * a.ld_dh)[c] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    __syncthreads();
  }
  // the rows that fill up the last k-block are contracted over with d = 0: they must be finite
  const int end = min(a.m, (all + BK - 1) / BK * BK);
  for (int r = all + static_cast<int>(blockIdx.x); r < end; r += gridDim.x)
    for (int c = tid; c < packets; c += kRowThreads)
      static_cast<uint4*>(a.hc)[static_cast<int64_t>(r) * packets + c] = make_uint4(0u, 0u, 0u, 0u);
}

// dh = unscale * sum over the splits for the counted rows. Four lanes share 8
// columns, each adding every fourth split in order, and are joined in order. 5-8
// us where dh is cut at all.
template <typename T>
__global__ void __launch_bounds__(256) ce_dh_finish(const float* __restrict__ acc, const RowHeader* header,
                                                    const int* __restrict__ row_index, int m, int k, int splits, T* dh,
                                                    int64_t ld_dh) {
  pdl_wait();
  pdl_trigger();
  const int64_t groups = static_cast<int64_t>(header->rows) * (k / 8);
  const float unscale = products_scale(header);
  const int part = threadIdx.x & 3;
  // all lanes of a warp take the same number of rounds: they exchange sums
  for (int64_t i0 = blockIdx.x * 64ll; i0 < groups; i0 += gridDim.x * 64ll) {
    const int64_t i = i0 + (threadIdx.x >> 2);
    const bool ok = i < groups;
    const int64_t row = ok ? i / (k / 8) : 0;
    const int col = ok ? static_cast<int>(i - row * (k / 8)) * 8 : 0;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = part; s < splits; s += 4) {
      const float4* src = reinterpret_cast<const float4*>(acc + (static_cast<int64_t>(s) * m + row) * k + col);
      const float4 a = __ldcs(src), b = __ldcs(src + 1);
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] += __shfl_xor_sync(0xffffffffu, v[e], 1);
      v[e] += __shfl_xor_sync(0xffffffffu, v[e], 2);
      v[e] *= unscale;
    }
    if (ok && part == 0) store8<T>(dh + row_index[row] * ld_dh + col, v);
  }
}

// ---- host side -------------------------------------------------------------------------

// Pairs of this kernel resident at once on the current device (each CTA takes
// a whole SM), asked once per device; 0 on failure.
template <int MODE, typename T, typename TW>
int resident_pairs(cudaLaunchConfig_t cfg) {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (cache[dev] == 0) {
    auto kern = ce_pair<MODE, T, TW>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(cfg.dynamicSmemBytes)) != cudaSuccess)
      return 0;
    cfg.gridDim = dim3(2, 1, 1);
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) != cudaSuccess) return 0;
    cache[dev] = clusters;
  }
  return cache[dev];
}

template <int MODE, typename T, typename TW>
int launch_pair(const char* what, const CeParams& p, int64_t tiles, int max_ctas, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = smem_of(MODE);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  int64_t pairs = resident_pairs<MODE, T, TW>(cfg);
  if (pairs <= 0)
    return fail(AXON_E_LAUNCH, "%s: no room for a CTA pair (%s)", what, cudaGetErrorString(cudaGetLastError()));
  if (max_ctas > 0 && max_ctas / 2 < pairs) pairs = max_ctas / 2 > 0 ? max_ctas / 2 : 1;
  if (tiles < pairs) pairs = tiles;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs), 1, 1);
  cudaError_t e = cudaLaunchKernelEx(&cfg, ce_pair<MODE, T, TW>, p);
  if (e != cudaSuccess) return fail(AXON_E_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return launch_status(what);
}

template <int MODE, typename T, int NT>
int launch_narrow_nt(const char* what, const CeParams& p, int grid, cudaStream_t s) {
  constexpr int smem = narrow_smem(MODE, NT);
  static bool set[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
    return fail(AXON_E_CUDA, "%s: no current device", what);
  auto kern = ce_narrow<MODE, T, NT>;
  if (!set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(AXON_E_LAUNCH, "%s: smem attribute: %s", what, cudaGetErrorString(e));
    set[dev] = true;
  }
  cudaError_t e = launch_k(kern, dim3(grid), dim3(narrow_threads(NT)), smem, s, p);
  if (e != cudaSuccess) return fail(AXON_E_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return launch_status(what);
}

// The rows a tile of ce_narrow holds.
int narrow_nt(int64_t m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128; }

template <int MODE, typename T>
int launch_narrow(const char* what, const CeParams& p, int grid, cudaStream_t s) {
  switch (narrow_nt(p.m)) {
    case 16: return launch_narrow_nt<MODE, T, 16>(what, p, grid, s);
    case 32: return launch_narrow_nt<MODE, T, 32>(what, p, grid, s);
    case 64: return launch_narrow_nt<MODE, T, 64>(what, p, grid, s);
    default: return launch_narrow_nt<MODE, T, 128>(what, p, grid, s);
  }
}

// Words a tile of ce_pair: the width, of 256 down to 128 in steps of 32, whose
// rounds of tiles take the least time (a k-block costs about 32 words more than
// its own): a narrower tile where the last round would be mostly empty (256 x
// 2048 x 32000: two rounds of 224 words instead of 256).
int wide_words(int64_t m, int64_t v) {
  const int64_t pairs = sm_count() / 2, row_tiles = (m + 255) / 256;
  int best = BN;
  int64_t least = INT64_MAX;
  for (int words = BN; words >= 128; words -= 32) {
    const int64_t rounds = (row_tiles * ((v + words - 1) / words) + pairs - 1) / pairs;
    if (rounds * (words + 32) < least) {
      least = rounds * (words + 32);
      best = words;
    }
  }
  return best;
}

// Words a tile of ce_narrow: the smallest multiple of 8 that needs no more
// rounds of tiles than 128 words would, so the last round is as full as the
// others (32000 words on 148 SMs: 286 tiles of 112 instead of 250 of 128).
int narrow_words(int64_t v, int max_ctas) {
  int64_t g = sm_count();
  if (max_ctas > 0 && max_ctas < g) g = max_ctas;
  const int64_t rounds = ((v + BM - 1) / BM + g - 1) / g;
  const int64_t words = (v + rounds * g - 1) / (rounds * g);
  return static_cast<int>((words + 7) / 8 * 8);
}

// CTAs of ce_narrow, at most one per SM.
int narrow_grid(int64_t v, int max_ctas) {
  const int64_t words = narrow_words(v, max_ctas), tiles = (v + words - 1) / words;
  int64_t g = sm_count();
  if (max_ctas > 0 && max_ctas < g) g = max_ctas;
  return static_cast<int>(tiles < g ? tiles : g);
}

int logits_words(int64_t m, int64_t v, int max_ctas) {
  return m > kNarrowRows ? wide_words(m, v) : narrow_words(v, max_ctas);
}

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Row tiles whose rows of h (512 k bytes a tile) take at most 48 MB: they stay
// in L2 beside the words that stream past.
int band_of(int64_t k) {
  const int64_t b = (48ll << 20) / (512 * k);
  return static_cast<int>(b < 1 ? 1 : b > 4096 ? 4096 : b);
}

// Rows of ce_few's dh tiles, or 0 where ce_pair works: more than 128 rows, or more
// blocks of 256 columns than CTAs (each keeps to one).
int few_rows(int64_t m, int64_t k, int max_ctas) {
  const int64_t grid = max_ctas > 0 && max_ctas < sm_count() ? max_ctas : sm_count();
  if (m > 128 || (k + BN - 1) / BN > grid) return 0;
  return m <= 32 ? 32 : m <= 64 ? 64 : 128;
}

struct GradPlan {
  int64_t piece;     // words a piece
  int64_t pieces;
  int splits;        // parts of dh's contraction over a piece
  int64_t off_rows, off_hc, off_d, off_acc, bytes;
};

constexpr int64_t kPieceBytes = 512ll << 20;  // of d

int layout(int64_t m, int64_t k, GradPlan& g) {
  g.off_rows = 256;
  g.off_hc = g.off_rows + round_up(5 * m * 4, 256);
  g.off_d = g.off_hc + round_up(m * k * 2, 256);
  g.off_acc = g.off_d + round_up(m * g.piece * 2, 256);
  g.bytes = g.off_acc + (g.pieces > 1 || g.splits > 1 ? round_up(g.splits * m * k * 4, 256) : 0);
  return AXON_OK;
}

int grad_plan(int64_t m, int64_t k, int64_t v, const axon_tune_t& t, GradPlan& g) {
  if (t.split < 0 || t.split % 256) return fail(AXON_E_ARG, "axon_linear_ce_grad: split must be a multiple of 256 words");
  if (t.split > 0) {
    g.piece = t.split;
  } else {
    int64_t most = kPieceBytes / (2 * (m ? m : 1)) / 256 * 256;
    if (most < 256) most = 256;
    const int64_t pieces = (v + most - 1) / most;
    g.piece = round_up((v + pieces - 1) / pieces, 256);
  }
  if (g.piece > round_up(v, 256)) g.piece = round_up(v, 256);
  g.pieces = (v + g.piece - 1) / g.piece;
  // A dh tile contracts over the whole piece while a dw tile contracts over the
  // rows: with few rows, few pairs would work on dh long after the rest. Cut
  // the contraction so that a part is at most a third of a pair's share, down
  // to 16 k-blocks and to what a dw tile takes. Uncut, the products of 64 x 2048
  // x 32000 took 174 us (103 cut, all else equal), of 1001 x 1024 x 50257 286 (170).
  const int64_t cols = (k + BN - 1) / BN, kb_dh = (g.piece + BK - 1) / BK, kb_dw = (m + BK - 1) / BK;
  if (few_rows(m, k, t.max_ctas)) {
    // ce_few: the number of parts (of 8 k-blocks at least) that leaves the SMs
    // the least uneven, among those that take each at most a few
    const int64_t tiles = (k + BM - 1) / BM, sms = sm_count();
    g.splits = 1;
    double least = 1e30;
    for (int64_t n = 1; n <= 3 * ((sms + tiles - 1) / tiles) && (n == 1 || kb_dh / n >= 8); ++n) {
      const double time = static_cast<double>((tiles * n + sms - 1) / sms) / n;
      if (time < least * 0.99) {
        least = time;
        g.splits = static_cast<int>(n);
      }
    }
    return layout(m, k, g);
  }
  const int64_t n_dh = (m + 255) / 256 * cols, n_dw = g.piece / 256 * cols;
  const int64_t pairs = sm_count() / 2;
  const int64_t share = (n_dh * (kb_dh + kTileCost) + n_dw * (kb_dw + kTileCost)) / pairs;
  int64_t part = share / 3 > 16 ? share / 3 : 16;
  if (part < kb_dw) part = kb_dw;
  if (part > kb_dh) part = kb_dh;
  g.splits = static_cast<int>((kb_dh + part - 1) / part);
  return layout(m, k, g);
}

int check_sizes(const char* what, int64_t m, int64_t k, int64_t v) {
  constexpr int64_t most = 1ll << 30;
  if (m < 0 || k < 1 || v < 1 || m > most || k > most || v > most)
    return fail(AXON_E_SHAPE, "%s: sizes out of range", what);
  if (k % 8) return fail(AXON_E_SHAPE, "%s: k must be a multiple of 8 (k=%lld)", what, (long long)k);
  return AXON_OK;
}

int check_head(const char* what, const void* h, const void* w, const void* targets, int64_t m, int64_t k, int64_t v,
               int64_t ld_h, int64_t ld_w, int32_t dtype, int32_t target_bits, int32_t reduction,
               const axon_tune_t& t) {
  int rc = check_sizes(what, m, k, v);
  if (rc) return rc;
  if (dtype != AXON_BF16 && dtype != AXON_F16)
    return fail(AXON_E_UNSUPPORTED, "%s: h and w must be bf16 or f16 (got %d)", what, dtype);
  if (target_bits != 32 && target_bits != 64)
    return fail(AXON_E_UNSUPPORTED, "%s: targets must be 32- or 64-bit integers", what);
  if (reduction < AXON_REDUCE_NONE || reduction > AXON_REDUCE_MEAN)
    return fail(AXON_E_ARG, "%s: unknown reduction %d", what, reduction);
  if (!w || (m > 0 && (!h || !targets))) return fail(AXON_E_ARG, "%s: NULL operand", what);
  if (ld_h < k || ld_w < k) return fail(AXON_E_SHAPE, "%s: leading dimension too small", what);
  if (ld_h % 8 || ld_w % 8) return fail(AXON_E_ALIGN, "%s: leading dimensions must be multiples of 8", what);
  if (!aligned16(h) || !aligned16(w)) return fail(AXON_E_ALIGN, "%s: operands must be 16-byte aligned", what);
  if (reinterpret_cast<uintptr_t>(targets) % (target_bits / 8))
    return fail(AXON_E_ALIGN, "%s: targets not aligned to their element", what);
  if (t.variant != 0) return fail(AXON_E_ARG, "%s: unknown variant %d", what, t.variant);
  if (t.max_ctas < 0) return fail(AXON_E_ARG, "%s: max_ctas must be >= 0", what);
  return AXON_OK;
}

// The operand maps of the logits: the wide kernel takes 128 rows of h and 128
// words a CTA, the narrow one 128 words and all rows.
int logits_maps(const char* what, CeParams& p, const void* h, int64_t ld_h, const void* w, int64_t ld_w, int32_t dtype) {
  int rc;
  if (p.m > kNarrowRows) {
    rc = make_map(&p.a, h, dtype, p.k, p.m, ld_h, BK, BM, "h", what);
    if (!rc) rc = make_map(&p.b, w, dtype, p.k, p.v, ld_w, BK, p.word_tile / 2, "w", what);
  } else {
    rc = make_map(&p.a, w, dtype, p.k, p.v, ld_w, BK, p.word_tile, "w", what);
    if (!rc) rc = make_map(&p.b, h, dtype, p.k, p.m, ld_h, BK, narrow_nt(p.m), "h", what);
  }
  p.a2 = p.c = p.a;  // not read by these modes (kDlogits' caller sets c)
  p.b2 = p.b;
  return rc;
}

template <int MODE, typename T>
int launch_logits(const char* what, const CeParams& p, int max_ctas, cudaStream_t s) {
  if (p.m <= kNarrowRows) return launch_narrow<MODE, T>(what, p, narrow_grid(p.v, max_ctas), s);
  const int64_t tiles = (p.m + 255ll) / 256 * ((p.v + p.word_tile - 1) / p.word_tile);
  return launch_pair<MODE, T, T>(what, p, tiles, max_ctas, s);
}

// Memory spans of an operand, [begin, end).
struct Span {
  const char* name;
  uintptr_t begin, end;
};

Span span(const char* name, const void* p, int64_t rows, int64_t ld, int64_t cols, int64_t item) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  return {name, at, p && rows > 0 ? at + static_cast<uintptr_t>(((rows - 1) * ld + cols) * item) : at};
}

// Outputs may overlap nothing: they are written while the operands are read.
int check_apart(const char* what, const Span* outs, int n_outs, const Span* ins, int n_ins) {
  for (int i = 0; i < n_outs; ++i) {
    for (int j = 0; j < n_ins; ++j)
      if (outs[i].begin < ins[j].end && ins[j].begin < outs[i].end)
        return fail(AXON_E_ARG, "%s: %s overlaps %s", what, outs[i].name, ins[j].name);
    for (int j = 0; j < i; ++j)
      if (outs[i].begin < outs[j].end && outs[j].begin < outs[i].end)
        return fail(AXON_E_ARG, "%s: %s overlaps %s", what, outs[i].name, outs[j].name);
  }
  return AXON_OK;
}

template <typename T>
int run_loss(const CeParams& p, const StatsArgs& a, int max_ctas, cudaStream_t s) {
  const char* what = "axon_linear_ce";
  int rc = launch_logits<kLse, T>(what, p, max_ctas, s);
  if (rc) return rc;
  launch_k(ce_stats<T>, dim3(static_cast<unsigned>((a.m + kStatsRows - 1) / kStatsRows)), dim3(kStatsThreads), 0, s, a);
  return launch_status(what);
}

template <int FEW, typename T, typename TW>
int launch_few_rows(const char* what, const CeParams& p, int grid, cudaStream_t s) {
  static bool set[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
    return fail(AXON_E_CUDA, "%s: no current device", what);
  auto kern = ce_few<FEW, T, TW>;
  if (!set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, few_smem(FEW));
    if (e != cudaSuccess) return fail(AXON_E_LAUNCH, "%s: smem attribute: %s", what, cudaGetErrorString(e));
    set[dev] = true;
  }
  cudaError_t e = launch_k(kern, dim3(grid), dim3(kFewThreads), few_smem(FEW), s, p);
  if (e != cudaSuccess) return fail(AXON_E_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return launch_status(what);
}

template <typename T, typename TW>
int launch_few(const char* what, const CeParams& p, int grid, cudaStream_t s) {
  switch (p.few) {
    case 32: return launch_few_rows<32, T, TW>(what, p, grid, s);
    case 64: return launch_few_rows<64, T, TW>(what, p, grid, s);
    default: return launch_few_rows<128, T, TW>(what, p, grid, s);
  }
}

// Both kernels of one piece.
template <typename T>
int run_piece(const CeParams& pl, const CeParams& pg, int32_t dw_dtype, int max_ctas, cudaStream_t s) {
  const char* what = "axon_linear_ce_grad";
  int rc = launch_logits<kDlogits, T>(what, pl, max_ctas, s);
  if (rc) return rc;
  if (pg.few) {
    int64_t grid = sm_count();
    if (max_ctas > 0 && max_ctas < grid) grid = max_ctas;
    return dw_dtype == AXON_F32 ? launch_few<T, float>(what, pg, static_cast<int>(grid), s)
                                : launch_few<T, T>(what, pg, static_cast<int>(grid), s);
  }
  const int64_t cols = (pg.k + BN - 1) / BN;
  const int64_t tiles = cols * ((pg.dh ? (pg.m + 255ll) / 256 * pg.splits : 0) + (pg.dw ? (pg.v + 255) / 256 : 0));
  if (dw_dtype == AXON_F32) return launch_pair<kGrads, T, float>(what, pg, tiles, max_ctas, s);
  return launch_pair<kGrads, T, T>(what, pg, tiles, max_ctas, s);
}

template <typename T>
int run_finish(const CeParams& p, cudaStream_t s) {
  const int64_t groups = static_cast<int64_t>(p.m) * (p.k / 8);
  const int64_t cap = 8ll * sm_count(), grid = (groups + 63) / 64;
  launch_k(ce_dh_finish<T>, dim3(static_cast<unsigned>(grid < cap ? grid : cap)), dim3(256), 0, s,
           static_cast<const float*>(p.acc), p.header, p.row_index, p.m, p.k, p.splits, static_cast<T*>(p.dh), p.ld_dh);
  return launch_status("axon_linear_ce_grad");
}

}  // namespace
}  // namespace axon

using namespace axon;

extern "C" {

int64_t axon_linear_ce_workspace_bytes(int64_t m, int64_t k, int64_t v) {
  int rc = check_sizes("axon_linear_ce", m, k, v);
  if (rc) return rc;
  const int64_t words = wide_words(m, v);
  return 256 + round_up(m * (m > kNarrowRows ? (v + words - 1) / words * 2 : sm_count()) * 8, 256);
}

int axon_linear_ce(const void* h, const void* w, const void* targets, float* lse, float* loss_rows, float* loss,
                   int64_t m, int64_t k, int64_t v, int64_t ld_h, int64_t ld_w, int32_t dtype, int32_t target_bits,
                   int64_t ignore_index, int32_t reduction, void* workspace, int64_t workspace_bytes,
                   const axon_tune_t* tune, void* stream) {
  return axon_linear_ce_kept(h, w, targets, lse, loss_rows, nullptr, loss, m, k, v, ld_h, ld_w, dtype, target_bits,
                             ignore_index, reduction, workspace, workspace_bytes, tune, stream);
}

int axon_linear_ce_kept(const void* h, const void* w, const void* targets, float* lse, float* loss_rows,
                        float* loss_copy, float* loss, int64_t m, int64_t k, int64_t v, int64_t ld_h, int64_t ld_w,
                        int32_t dtype, int32_t target_bits, int64_t ignore_index, int32_t reduction, void* workspace,
                        int64_t workspace_bytes, const axon_tune_t* tune, void* stream) {
  const char* what = "axon_linear_ce";
  axon_tune_t t = tune_or_default(tune);
  int rc = check_head(what, h, w, targets, m, k, v, ld_h, ld_w, dtype, target_bits, reduction, t);
  if (rc) return rc;
  if (m > 0 && (!lse || !loss_rows)) return fail(AXON_E_ARG, "%s: NULL output", what);
  if (reduction != AXON_REDUCE_NONE && !loss) return fail(AXON_E_ARG, "%s: NULL loss", what);
  const int64_t need = axon_linear_ce_workspace_bytes(m, k, v);
  if (m > 0 && (!workspace || workspace_bytes < need))
    return fail(AXON_E_ARG, "%s: workspace of %lld bytes needed", what, (long long)need);
  if (!aligned16(workspace)) return fail(AXON_E_ALIGN, "%s: workspace must be 16-byte aligned", what);
  cudaStream_t s = as_stream(stream);
  if (m == 0) {  // no rows: a sum of nothing, a mean of nothing
    if (reduction == AXON_REDUCE_NONE) return AXON_OK;
    cudaError_t e = cudaMemsetAsync(loss, reduction == AXON_REDUCE_MEAN ? 0xff : 0, sizeof(float), s);
    return e == cudaSuccess ? AXON_OK : fail(AXON_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  CeParams p{};
  p.m = static_cast<int>(m);
  p.v = static_cast<int>(v);
  p.k = static_cast<int>(k);
  p.targets = targets;
  p.target64 = target_bits == 64;
  p.ignore_index = ignore_index;
  p.done = static_cast<unsigned*>(workspace);
  p.part = reinterpret_cast<float2*>(static_cast<char*>(workspace) + 256);
  p.word_tile = logits_words(m, v, t.max_ctas);
  p.parts = static_cast<int>(m > kNarrowRows ? (v + p.word_tile - 1) / p.word_tile * 2 : narrow_grid(v, t.max_ctas));
  p.band = band_of(k);
  if ((rc = logits_maps(what, p, h, ld_h, w, ld_w, dtype))) return rc;
  const StatsArgs a{h, w, ld_h, ld_w, p.part, targets, p.target64, ignore_index, p.m, p.k, p.v, p.parts, lse, loss_rows,
                    loss_copy, reduction == AXON_REDUCE_NONE ? nullptr : loss, reduction == AXON_REDUCE_MEAN, p.done};
  return dtype == AXON_BF16 ? run_loss<__nv_bfloat16>(p, a, t.max_ctas, s) : run_loss<__half>(p, a, t.max_ctas, s);
}

int64_t axon_linear_ce_grad_workspace_bytes(int64_t m, int64_t k, int64_t v, const axon_tune_t* tune) {
  int rc = check_sizes("axon_linear_ce_grad", m, k, v);
  if (rc) return rc;
  GradPlan g;
  rc = grad_plan(m, k, v, tune_or_default(tune), g);
  return rc ? rc : g.bytes;
}

int axon_linear_ce_grad(const void* h, const void* w, const void* targets, const float* lse, const float* loss_rows,
                        const float* dloss, void* dh, void* dw, int64_t m, int64_t k, int64_t v, int64_t ld_h,
                        int64_t ld_w, int64_t ld_dh, int64_t ld_dw, int32_t dtype, int32_t dw_dtype,
                        int32_t target_bits, int64_t ignore_index, int32_t reduction, void* workspace,
                        int64_t workspace_bytes, const axon_tune_t* tune, void* stream) {
  const char* what = "axon_linear_ce_grad";
  axon_tune_t t = tune_or_default(tune);
  int rc = check_head(what, h, w, targets, m, k, v, ld_h, ld_w, dtype, target_bits, reduction, t);
  if (rc) return rc;
  if (dw_dtype != dtype && dw_dtype != AXON_F32)
    return fail(AXON_E_UNSUPPORTED, "%s: dw must have w's type or fp32 (got %d)", what, dw_dtype);
  if (m > 0 && (!lse || !loss_rows || !dloss)) return fail(AXON_E_ARG, "%s: NULL operand", what);
  if (m > 0 && !dh && !dw) return fail(AXON_E_ARG, "%s: dh and dw are both NULL", what);
  if ((dh && ld_dh < k) || (dw && ld_dw < k)) return fail(AXON_E_SHAPE, "%s: leading dimension too small", what);
  if ((dh && ld_dh % 8) || (dw && ld_dw % 8))
    return fail(AXON_E_ALIGN, "%s: leading dimensions must be multiples of 8", what);
  if (!aligned16(dh) || !aligned16(dw)) return fail(AXON_E_ALIGN, "%s: outputs must be 16-byte aligned", what);
  const Span outs[2] = {span("dh", dh, m, ld_dh, k, 2), span("dw", dw, v, ld_dw, k, dtype_size(dw_dtype))};
  const Span ins[6] = {span("h", h, m, ld_h, k, 2),   span("w", w, v, ld_w, k, 2),
                       span("targets", targets, m, 1, 1, target_bits / 8), span("lse", lse, m, 1, 1, 4),
                       span("loss_rows", loss_rows, m, 1, 1, 4),
                       span("dloss", dloss, reduction == AXON_REDUCE_NONE ? m : 1, 1, 1, 4)};
  if ((rc = check_apart(what, outs, 2, ins, 6))) return rc;
  cudaStream_t s = as_stream(stream);
  if (m == 0) {  // no rows: dw is zero
    if (!dw) return AXON_OK;
    cudaError_t e = cudaMemset2DAsync(dw, ld_dw * dtype_size(dw_dtype), 0, k * dtype_size(dw_dtype), v, s);
    return e == cudaSuccess ? AXON_OK : fail(AXON_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  GradPlan g;
  if ((rc = grad_plan(m, k, v, t, g))) return rc;
  if (!workspace || workspace_bytes < g.bytes)
    return fail(AXON_E_ARG, "%s: workspace of %lld bytes needed", what, (long long)g.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) & 255u)
    return fail(AXON_E_ALIGN, "%s: workspace must be 256-byte aligned", what);
  char* ws = static_cast<char*>(workspace);
  RowsArgs ra{};
  ra.h = h;
  ra.ld_h = ld_h;
  ra.targets = targets;
  ra.target64 = target_bits == 64;
  ra.ignore_index = ignore_index;
  ra.v = v;
  ra.lse = lse;
  ra.loss = loss_rows;
  ra.dloss = dloss;
  ra.per_row = reduction == AXON_REDUCE_NONE;
  ra.mean = reduction == AXON_REDUCE_MEAN;
  ra.f16 = dtype == AXON_F16;
  ra.m = static_cast<int>(m);
  ra.k = static_cast<int>(k);
  ra.dh = dh;
  ra.ld_dh = ld_dh;
  ra.header = reinterpret_cast<RowHeader*>(ws);
  ra.row_index = reinterpret_cast<int*>(ws + g.off_rows);
  ra.row_target = ra.row_index + m;
  ra.row_lse = reinterpret_cast<float*>(ra.row_target + m);
  ra.row_g = ra.row_lse + m;
  ra.row_dt = ra.row_g + m;
  ra.hc = ws + g.off_hc;
  const int64_t cap = 4ll * sm_count();
  launch_k(ce_grad_rows, dim3(static_cast<unsigned>(m < cap ? m : cap)), dim3(kRowThreads), 0, s, ra);
  if ((rc = launch_status(what))) return rc;

  for (int64_t i = 0; i < g.pieces; ++i) {
    const int64_t v0 = i * g.piece, vc = v - v0 < g.piece ? v - v0 : g.piece;
    const char* wp = static_cast<const char*>(w) + v0 * ld_w * 2;
    CeParams p{};
    p.m = static_cast<int>(m);
    p.v = static_cast<int>(vc);
    p.k = static_cast<int>(k);
    p.header = ra.header;
    p.row_target = ra.row_target;
    p.row_lse = ra.row_lse;
    p.row_g = ra.row_g;
    p.row_dt = ra.row_dt;
    p.row_index = ra.row_index;
    p.v0 = static_cast<int>(v0);
    p.d = ws + g.off_d;
    p.ld_d = round_up(vc, 8);
    p.dh = dh;
    p.dw = dw;
    p.ld_dh = ld_dh;
    p.acc = reinterpret_cast<float*>(ws + g.off_acc);
    p.first = i == 0;
    p.last = i + 1 == g.pieces;
    p.band = band_of(k);
    p.splits = g.splits;
    p.word_tile = logits_words(m, vc, t.max_ctas);
    CeParams pg = p;
    if ((rc = logits_maps(what, p, ra.hc, k, wp, ld_w, dtype))) return rc;
    if ((rc = make_map(&p.c, p.d, dtype, vc, m, p.ld_d, 64, 32, "d", what))) return rc;
    pg.few = few_rows(m, k, t.max_ctas);
    if ((rc = make_map(&pg.a, p.d, dtype, vc, m, p.ld_d, BK, pg.few ? pg.few : BM, "d", what))) return rc;
    if ((rc = make_map(&pg.b, wp, dtype, k, vc, ld_w, 64, BK, "w", what))) return rc;
    if ((rc = make_map(&pg.a2, p.d, dtype, vc, m, p.ld_d, 64, BK, "d", what))) return rc;
    if ((rc = make_map(&pg.b2, ra.hc, dtype, k, m, k, 64, BK, "h", what))) return rc;
    pg.c = pg.a;
    if (dw) {
      char* dwp = static_cast<char*>(dw) + v0 * ld_dw * dtype_size(dw_dtype);
      if ((rc = make_map(&pg.c, dwp, dw_dtype, k, vc, ld_dw, 128 / dtype_size(dw_dtype), 32, "dw", what))) return rc;
    }
    rc = dtype == AXON_BF16 ? run_piece<__nv_bfloat16>(p, pg, dw_dtype, t.max_ctas, s)
                            : run_piece<__half>(p, pg, dw_dtype, t.max_ctas, s);
    if (rc) return rc;
    if (p.last && dh && g.splits > 1 &&
        (rc = dtype == AXON_BF16 ? run_finish<__nv_bfloat16>(p, s) : run_finish<__half>(p, s)))
      return rc;
  }
  return AXON_OK;
}

int axon_selftest_linear_ce_gave_up(void* stream) {
  const int code = AXON_E_TIMEOUT;
  cudaStream_t s = as_stream(stream);
  cudaError_t e = cudaMemcpyToSymbolAsync(g_ce_error, &code, sizeof(int), 0, cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  return e == cudaSuccess ? AXON_OK : fail(AXON_E_CUDA, "axon_selftest_linear_ce_gave_up: %s", cudaGetErrorString(e));
}

int axon_linear_ce_status(void* stream) {
  int v = 0;
  cudaStream_t s = as_stream(stream);
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_ce_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return fail(AXON_E_CUDA, "axon_linear_ce_status: %s", cudaGetErrorString(e));
  if (v != 0) {
    int zero = 0;
    cudaMemcpyToSymbolAsync(g_ce_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s);
    cudaStreamSynchronize(s);
    return fail(v, "axon_linear_ce: a pipeline wait gave up (status %d)", v);
  }
  return AXON_OK;
}

}  // extern "C"
