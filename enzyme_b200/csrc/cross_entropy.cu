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
//             k = 4096), is a dot product of its own in fp32 lanes.
//   kDlogits  a piece of the vocabulary at a time, s is formed again and leaves as
//             d, rounded to the operand type, in the workspace [rows, piece].
//             The target's entry is g (p_t - 1) = g expm1(-loss).
//   kGrads    both products of d for that piece in one launch: tiles of dh (d as
//             it lies, contracted over the piece, added to an fp32 accumulator
//             until the last piece) and tiles of dw (d transposed, taken by TMA as
//             an MN-major A operand, contracted over the rows).
//
// The gradient works on the rows that count: ce_grad_rows moves them to the
// front (a copy of h, a few microseconds) and hands the later kernels their
// number on the device, so ignored rows cost nothing and whatever they hold
// (NaN, infinities) reaches nothing.
//
// f16: d is held times a power of two that puts the largest |g| near 2^14, so
// that small probabilities are not lost below 2^-24; the epilogues undo it.
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
constexpr int kStages = 7;           // 7 x 32 KB of the 227 KB
constexpr uint32_t TMEM_COLS = 2 * BN;
constexpr float kLog2e = 1.4426950408889634f;

enum Mode { kLse = 0, kDlogits = 1, kGrads = 2 };

// What ce_grad_rows hands to the kernels after it.
struct RowHeader {
  int rows;         // rows that count
  float unscale;    // 1 / the power of two that d carries
};

struct CeParams {
  CUtensorMap a, b;     // kLse, kDlogits: h, w.   kGrads, dh tiles: d, w's piece
  CUtensorMap a2, b2;   // kGrads, dw tiles: d transposed, h
  int m, v, k;          // rows (at most), words of this piece, hidden size
  const RowHeader* header;  // NULL: all m rows
  // kLse
  const void* targets;
  int target64;
  int64_t ignore_index;
  float2* part;         // [m][word tiles]
  // kDlogits: per counted row
  const int* row_target;
  const float* row_lse;
  const float* row_g;
  const float* row_dt;
  int v0;               // first word of the piece
  void* d;              // [rows rounded up to 256][ld_d]
  int64_t ld_d;
  // kGrads
  const int* row_index; // counted row -> row of dh
  void* dh;
  void* dw;
  int64_t ld_dh, ld_dw;
  float* acc;           // fp32 [rows rounded up][k] between pieces
  int first, last;      // this piece is the vocabulary's first / last
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

// exp(x - ref)
__device__ __forceinline__ float exp_from(float x, float ref) { return ex2((x - ref) * kLog2e); }

// ---- tiles -----------------------------------------------------------------------------

struct Tile {
  bool dw;          // kGrads: a tile of dw (else of dh)
  int tm, tn, kb;   // row tile, column tile, k-blocks
};

struct Walk {
  int pair, pairs, rows;
};

// The `i`-th tile of this pair; false past the last one.
//
// kLse, kDlogits: bands of `band` row tiles (so that a band of h stays in L2),
// each band word tile by word tile.
//
// kGrads: dh tiles (a contraction over the whole piece) first, dealt in turn;
// the pairs that got one fewer start their dw tiles earlier, by as many as fit
// in one dh tile's time, and the rest of the dw tiles is dealt in turn. Row
// tiles run fastest for dh and column tiles for dw, so that the pairs share
// the words, then d, in L2.
template <int MODE>
__device__ __forceinline__ bool tile_at(const CeParams& p, const Walk& w, int i, Tile& t) {
  const int row_tiles = (w.rows + 2 * BM - 1) / (2 * BM);
  if constexpr (MODE != kGrads) {
    const int word_tiles = (p.v + BN - 1) / BN;
    const int64_t at = static_cast<int64_t>(i) * w.pairs + w.pair;
    if (at >= static_cast<int64_t>(row_tiles) * word_tiles) return false;
    const int64_t per_band = static_cast<int64_t>(p.band) * word_tiles;
    const int band = static_cast<int>(at / per_band);
    const int64_t within = at - band * per_band;
    const int rows = row_tiles - band * p.band < p.band ? row_tiles - band * p.band : p.band;
    t.dw = false;
    t.tm = band * p.band + static_cast<int>(within % rows);
    t.tn = static_cast<int>(within / rows);
    t.kb = (p.k + BK - 1) / BK;
    return true;
  } else {
    const int col_tiles = (p.k + BN - 1) / BN;
    const int word_tiles = (p.v + 2 * BM - 1) / (2 * BM);
    const int n_dh = p.dh ? row_tiles * col_tiles : 0;
    const int n_dw = p.dw ? word_tiles * col_tiles : 0;
    const int kb_dh = (p.v + BK - 1) / BK, kb_dw = (w.rows + BK - 1) / BK;
    const int odd = n_dh % w.pairs;  // pairs below this one have a dh tile more
    const int mine = n_dh / w.pairs + (w.pair < odd ? 1 : 0);
    int at;
    if (i < mine) {
      at = i * w.pairs + w.pair;
      t.dw = false;
      t.tm = at % row_tiles;
      t.tn = at / row_tiles;
      t.kb = kb_dh;
      return true;
    }
    i -= mine;
    const int behind = odd ? w.pairs - odd : 0;  // pairs with one dh tile fewer
    int early = kb_dw > 0 ? kb_dh / kb_dw : 0;   // dw tiles they take meanwhile
    if (behind && early > n_dw / behind) early = n_dw / behind;
    if (behind && w.pair >= odd) {
      if (i < early) {
        at = i * behind + (w.pair - odd);
        t.dw = true;
        t.tm = at / col_tiles;
        t.tn = at % col_tiles;
        t.kb = kb_dw;
        return true;
      }
      i -= early;
    }
    const int64_t rest = static_cast<int64_t>(behind) * early + static_cast<int64_t>(i) * w.pairs + w.pair;
    if (rest >= n_dw) return false;
    t.dw = true;
    t.tm = static_cast<int>(rest / col_tiles);
    t.tn = static_cast<int>(rest % col_tiles);
    t.kb = kb_dw;
    return true;
  }
}

// One k-block of this CTA's half of the operands: 128 rows of A, 128 columns
// of B, 32 KB. K-major operands come as 128 rows x 64 elements of k; MN-major
// ones as two blocks of 64 elements x 64 rows of k.
template <int MODE>
__device__ __forceinline__ void load_stage(const CeParams& p, const Tile& t, int kb, int rank, uint8_t* sa,
                                           uint32_t full) {
  uint8_t* sb = sa + A_BYTES;
  const int row0 = t.tm * 2 * BM + rank * BM;
  const int col0 = t.tn * BN + rank * BH;
  if constexpr (MODE != kGrads) {
    tma_load_2d_pair(&p.a, full, sa, kb * BK, row0);
    tma_load_2d_pair(&p.b, full, sb, kb * BK, col0);
  } else {
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

// tcgen05 instruction descriptor: fp32 accumulator, M 256, N 256; bit 15 / 16:
// A / B is MN-major.
template <typename T>
__device__ __forceinline__ uint32_t idesc(bool a_mn, bool b_mn) {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>((2 * BM) >> 4) << 24);
}

// ---- epilogues -----------------------------------------------------------------------

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

// kLse: this thread's row over the tile's words.
__device__ __forceinline__ void lse_tile(const CeParams& p, const Tile& t, uint32_t tbase, int64_t row, bool row_ok) {
  const float ninf = __int_as_float(0xff800000);
  const int target = row_ok ? load_target(p.targets, p.target64, row, p.ignore_index, p.v) : -1;
  float mx = ninf, sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    const int col = t.tn * BN + c * 32;
    if (col >= p.v) break;  // the same for the whole warp
    float v[32];
    __syncwarp();
    tmem_ld32(tbase + c * 32, v);
    tmem_wait_ld();
    if (col + 32 > p.v) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col + j >= p.v) v[j] = ninf;
    }
    if (target >= col && target < col + 32) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (target == col + j) v[j] = ninf;
    }
    const float nm = fmaxf(mx, max32(v));
    const float ref = nm == ninf ? 0.f : nm;  // nothing counted yet: exp gives 0
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 32; ++j) s[j & 3] += exp_from(v[j], ref);
    sum = sum * exp_from(mx, ref) + ((s[0] + s[1]) + (s[2] + s[3]));
    mx = nm;
  }
  if (row_ok) p.part[row * ((p.v + BN - 1) / BN) + t.tn] = make_float2(mx, sum);
}

template <typename T>
__device__ __forceinline__ void store32_full(T* dst, const float* v) {
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    Vec<T> pk;
#pragma unroll
    for (int e = 0; e < 8; ++e) pk.e[e] = from_f<T>(v[j + e]);
    st_vec(dst + j, pk);
  }
}

// kDlogits: d for this thread's row. Rows past the counted ones inside the
// tile are written as zeros (the contraction over rows reads them), and so
// are the words that pad ld_d.
template <typename T>
__device__ __forceinline__ void dlogits_tile(const CeParams& p, const Tile& t, uint32_t tbase, int64_t row,
                                             bool row_ok) {
  const float lse = row_ok ? p.row_lse[row] : 0.f;
  const float g = row_ok ? p.row_g[row] : 0.f;
  const int target = row_ok ? p.row_target[row] - p.v0 : -1;
  T* drow = static_cast<T*>(p.d) + row * p.ld_d;
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    const int col = t.tn * BN + c * 32;
    if (col >= p.v) break;
    float v[32];
    __syncwarp();
    tmem_ld32(tbase + c * 32, v);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = row_ok && col + j < p.v ? exp_from(v[j], lse) * g : 0.f;
    if (target >= col && target < col + 32) {
      const float dt = p.row_dt[row];
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (target == col + j) v[j] = dt;
    }
    if (col + 32 <= p.ld_d) {
      store32_full<T>(drow + col, v);
    } else {
#pragma unroll
      for (int j = 0; j < 32; j += 8)
        if (col + j < p.ld_d) {
          Vec<T> pk;
#pragma unroll
          for (int e = 0; e < 8; ++e) pk.e[e] = from_f<T>(v[j + e]);
          st_vec(drow + col + j, pk);
        }
    }
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

// kGrads: this thread's row of a tile of dh or dw.
template <typename T, typename TW>
__device__ __forceinline__ void grad_tile(const CeParams& p, const Walk& w, const Tile& t, uint32_t tbase, int64_t row,
                                          float unscale) {
  const bool row_ok = t.dw ? row < p.v : row < w.rows;
  const int64_t out_row = row_ok ? (t.dw ? p.v0 + row : (p.last ? p.row_index[row] : 0)) : 0;
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    const int col = t.tn * BN + c * 32;
    if (col >= p.k) break;
    float v[32];
    __syncwarp();
    tmem_ld32(tbase + c * 32, v);
    tmem_wait_ld();
    if (!row_ok) continue;
    if (t.kb == 0) {  // no row counts: the accumulator was never written
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      if (col + j >= p.k) break;  // k is a multiple of 8
      if (t.dw) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j + e] *= unscale;
        store8<TW>(static_cast<TW*>(p.dw) + out_row * p.ld_dw + col + j, v + j);
        continue;
      }
      float* acc = p.acc + row * p.k + col + j;
      if (!p.first) {
        const float4 a = *reinterpret_cast<const float4*>(acc), b = *reinterpret_cast<const float4*>(acc + 4);
        v[j] += a.x; v[j + 1] += a.y; v[j + 2] += a.z; v[j + 3] += a.w;
        v[j + 4] += b.x; v[j + 5] += b.y; v[j + 6] += b.z; v[j + 7] += b.w;
      }
      if (p.last) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j + e] *= unscale;
        store8<T>(static_cast<T*>(p.dh) + out_row * p.ld_dh + col + j, v + j);
      } else {
        store8<float>(acc, v + j);
      }
    }
  }
}

// ---- the CTA-pair kernel ---------------------------------------------------------------

template <int MODE, typename T, typename TW>
__global__ void __launch_bounds__(192, 1) ce_pair(const __grid_constant__ CeParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * STAGE);
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
      mbar_init(&tempty[b], 8);  // one arrival per epilogue warp of each CTA
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

  Walk w;
  w.pair = blockIdx.x >> 1;
  w.pairs = gridDim.x >> 1;
  w.rows = p.header ? p.header->rows : p.m;
  Tile t;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; tile_at<MODE>(p, w, i, t); ++i) {
      for (int kb = 0; kb < t.kb; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, &g_ce_error)) goto producer_done;
        const uint32_t leader_full = mapa_u32(smem_u32(&full[stage]), 0);
        if (leader) mbar_expect_tx(&full[stage], 2 * STAGE);
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
    for (int i = 0; tile_at<MODE>(p, w, i, t); ++i) {
      const int buf = i & 1;
      if (!mbar_wait(&tempty[buf], ((i >> 1) & 1) ^ 1u, abort_flag, &g_ce_error)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + static_cast<uint32_t>(buf * BN);
      const bool a_mn = MODE == kGrads && t.dw, b_mn = MODE == kGrads;
      const uint32_t id = idesc<T>(a_mn, b_mn);
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
    const float unscale = MODE == kGrads ? p.header->unscale : 1.f;
    for (int i = 0; tile_at<MODE>(p, w, i, t); ++i) {
      const int buf = i & 1;
      if (!mbar_wait(&tfull[buf], (i >> 1) & 1, abort_flag, &g_ce_error)) break;
      tc_fence_after();
      const int64_t row = static_cast<int64_t>(t.tm) * 2 * BM + rank * BM + q * 32 + lane;
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(buf * BN);
      if constexpr (MODE == kLse) lse_tile(p, t, tbase, row, row < w.rows);
      else if constexpr (MODE == kDlogits) dlogits_tile<T>(p, t, tbase, row, row < w.rows);
      else grad_tile<T, TW>(p, w, t, tbase, row, unscale);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(&tempty[buf]), 0), 1);
    }
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

struct StatsArgs {
  const void* h;
  const void* w;
  int64_t ld_h, ld_w;
  const float2* part;
  const void* targets;
  int target64;
  int64_t ignore_index;
  int m, k, v, tiles;
  float* lse;
  float* loss;
};

// Joins a row's (max, sum) of every word tile with the target's logit, a warp
// per row.
template <typename T>
__global__ void __launch_bounds__(128) ce_stats(StatsArgs a) {
  const float ninf = __int_as_float(0xff800000);
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= a.m) return;
  const int target = load_target(a.targets, a.target64, row, a.ignore_index, a.v);
  float at = 0.f;
  if (target >= 0)
    at = warp_dot(static_cast<const T*>(a.h) + row * a.ld_h, static_cast<const T*>(a.w) + target * a.ld_w, a.k, lane);
  const float2* pr = a.part + row * a.tiles;
  float mx = ninf;
  for (int i = lane; i < a.tiles; i += 32) mx = fmaxf(mx, pr[i].x);
  mx = warp_max(mx);
  const float ref = mx == ninf ? 0.f : mx;
  float sum = 0.f;
  for (int i = lane; i < a.tiles; i += 32) {
    const float2 t = pr[i];
    sum += t.y * exp_from(t.x, ref);
  }
  sum = warp_sum(sum);
  if (lane) return;
  // the log-sum-exp over the words other than the target, and the loss, in 64
  // bits: a row each, and an almost certain target leaves a loss far below
  // the logits' own rounding
  const double rest = static_cast<double>(ref) + log(static_cast<double>(sum));
  double lse = rest, loss = 0.0;
  if (target >= 0) {
    const double st = at;
    const double x = rest - st;
    loss = x > 0.0 ? x + log1p(exp(-x)) : log1p(exp(x));
    lse = x > 0.0 ? rest + log1p(exp(-x)) : st + loss;
    if (st > 3.5e38) loss = lse - st;  // an infinite logit: NaN, as lse - s_t says, not 0
  } else if (target == -2) {
    loss = __longlong_as_double(0x7ff8000000000000ll);
  }
  a.lse[row] = static_cast<float>(lse);
  a.loss[row] = static_cast<float>(loss);
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

// Sum or mean of the rows' losses: one CTA, float64, fixed order.
__global__ void __launch_bounds__(1024) ce_reduce(const float* __restrict__ loss_rows, const void* targets, int target64,
                                                  int64_t ignore_index, int64_t v, int m, int mean, float* loss) {
  double sum = 0.0;
  int count = 0;
  for (int i = threadIdx.x; i < m; i += 1024) {
    sum += static_cast<double>(loss_rows[i]);
    count += load_target(targets, target64, i, ignore_index, v) != -1;
  }
  sum = cta_sum<double, 1024>(sum);
  count = cta_sum<int, 1024>(count);
  if (threadIdx.x == 0) *loss = static_cast<float>(mean ? sum / static_cast<double>(count) : sum);
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
  void* hc;           // [m rounded up to 256][k]
};

constexpr int kRowThreads = 256;

// Moves the rows that count to the front. Every CTA owns a range of rows; it
// finds the number of counted rows before its own (and, for f16, the largest
// |g|) by reading all targets itself: m is at most some ten thousands, and a
// second launch would cost more.
__global__ void __launch_bounds__(kRowThreads) ce_grad_rows(RowsArgs a) {
  __shared__ int slot[kRowThreads];
  __shared__ int warp_count[kRowThreads / 32];
  __shared__ float warp_top[kRowThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.m + gridDim.x - 1) / gridDim.x;
  const int r0 = min(a.m, static_cast<int>(blockIdx.x) * per), r1 = min(a.m, r0 + per);
  int before = 0, all = 0;
  float top = 0.f;
  for (int i = tid; i < a.m; i += kRowThreads) {
    if (load_target(a.targets, a.target64, i, a.ignore_index, a.v) == -1) continue;
    all += 1;
    before += i < r0;
    if (a.f16) top = fmaxf(top, fabsf(a.dloss[a.per_row ? i : 0]));
  }
  before = cta_sum<int, kRowThreads>(before);
  all = cta_sum<int, kRowThreads>(all);
  float scale = 1.f;
  if (a.f16) {
    top = warp_max(top);
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
    for (int i = 0; i < kRowThreads / 32; ++i) top = fmaxf(top, warp_top[i]);
    if (a.mean) top /= static_cast<float>(all);
    if (top > 0.f && top < __int_as_float(0x7f800000)) {
      // 2^(14 - floor(log2 top)), kept where it and its inverse are normal numbers
      int e = 14 - ilogbf(top);
      e = max(-126, min(126, e));
      scale = ldexpf(1.f, e);
    }
  }
  if (blockIdx.x == 0 && tid == 0) *a.header = RowHeader{all, 1.f / scale};

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
      if (a.mean) g /= static_cast<float>(all);
      if (target == -2) g = __int_as_float(0x7fc00000);  // a target outside the vocabulary poisons the gradients
      g *= scale;
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
  // the rows that fill up the last row tile are contracted over with d = 0: they must be finite
  const int end = (all + 255) / 256 * 256;
  for (int r = all + static_cast<int>(blockIdx.x); r < end; r += gridDim.x)
    for (int c = tid; c < packets; c += kRowThreads)
      static_cast<uint4*>(a.hc)[static_cast<int64_t>(r) * packets + c] = make_uint4(0u, 0u, 0u, 0u);
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
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(192, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(kStages) * STAGE + 1024 + 256;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
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

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Row tiles whose rows of h (512 k bytes a tile) take at most 48 MB: they stay
// in L2 beside the words that stream past.
int band_of(int64_t k) {
  const int64_t b = (48ll << 20) / (512 * k);
  return static_cast<int>(b < 1 ? 1 : b > 4096 ? 4096 : b);
}

struct GradPlan {
  int64_t rows;      // m rounded up to the row tile
  int64_t piece;     // words a piece
  int64_t pieces;
  int64_t off_rows, off_hc, off_d, off_acc, bytes;
};

constexpr int64_t kPieceBytes = 512ll << 20;  // of d

int grad_plan(int64_t m, int64_t k, int64_t v, const axon_tune_t& t, GradPlan& g) {
  g.rows = round_up(m, 256);
  if (t.split < 0 || t.split % 256) return fail(AXON_E_ARG, "axon_linear_ce_grad: split must be a multiple of 256 words");
  if (t.split > 0) {
    g.piece = t.split;
  } else {
    int64_t most = kPieceBytes / (2 * (g.rows ? g.rows : 256)) / 256 * 256;
    if (most < 256) most = 256;
    const int64_t pieces = (v + most - 1) / most;
    g.piece = round_up((v + pieces - 1) / pieces, 256);
  }
  if (g.piece > round_up(v, 256)) g.piece = round_up(v, 256);
  g.pieces = (v + g.piece - 1) / g.piece;
  g.off_rows = 256;
  g.off_hc = g.off_rows + round_up(5 * g.rows * 4, 256);
  g.off_d = g.off_hc + round_up(g.rows * k * 2, 256);
  g.off_acc = g.off_d + round_up(g.rows * g.piece * 2, 256);
  g.bytes = g.off_acc + (g.pieces > 1 ? round_up(g.rows * k * 4, 256) : 0);
  return AXON_OK;
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

template <typename T>
int run_loss(const CeParams& p, int64_t tiles, int max_ctas, cudaStream_t s) {
  return launch_pair<kLse, T, T>("axon_linear_ce", p, tiles, max_ctas, s);
}

// Both kernels of one piece.
template <typename T>
int run_piece(const CeParams& pl, const CeParams& pg, int32_t dw_dtype, int64_t rows, int max_ctas, cudaStream_t s) {
  const char* what = "axon_linear_ce_grad";
  int rc = launch_pair<kDlogits, T, T>(what, pl, rows / 256 * ((pl.v + BN - 1) / BN), max_ctas, s);
  if (rc) return rc;
  const int64_t cols = (pg.k + BN - 1) / BN;
  const int64_t tiles = cols * ((pg.dh ? rows / 256 : 0) + (pg.dw ? (pg.v + 255) / 256 : 0));
  if (dw_dtype == AXON_F32) return launch_pair<kGrads, T, float>(what, pg, tiles, max_ctas, s);
  return launch_pair<kGrads, T, T>(what, pg, tiles, max_ctas, s);
}

}  // namespace
}  // namespace axon

using namespace axon;

extern "C" {

int64_t axon_linear_ce_workspace_bytes(int64_t m, int64_t k, int64_t v) {
  int rc = check_sizes("axon_linear_ce", m, k, v);
  if (rc) return rc;
  return round_up(m * ((v + BN - 1) / BN) * 8, 256) + 256;
}

int axon_linear_ce(const void* h, const void* w, const void* targets, float* lse, float* loss_rows, float* loss,
                   int64_t m, int64_t k, int64_t v, int64_t ld_h, int64_t ld_w, int32_t dtype, int32_t target_bits,
                   int64_t ignore_index, int32_t reduction, void* workspace, int64_t workspace_bytes,
                   const axon_tune_t* tune, void* stream) {
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
  const int64_t word_tiles = (v + BN - 1) / BN;
  if (m > 0) {
    CeParams p{};
    if ((rc = make_map(&p.a, h, dtype, k, m, ld_h, BK, BM, "h", what))) return rc;
    if ((rc = make_map(&p.b, w, dtype, k, v, ld_w, BK, BH, "w", what))) return rc;
    p.a2 = p.a;
    p.b2 = p.b;
    p.m = static_cast<int>(m);
    p.v = static_cast<int>(v);
    p.k = static_cast<int>(k);
    p.targets = targets;
    p.target64 = target_bits == 64;
    p.ignore_index = ignore_index;
    p.part = static_cast<float2*>(workspace);
    p.band = band_of(k);
    const int64_t tiles = (m + 255) / 256 * word_tiles;
    rc = dtype == AXON_BF16 ? run_loss<__nv_bfloat16>(p, tiles, t.max_ctas, s) : run_loss<__half>(p, tiles, t.max_ctas, s);
    if (rc) return rc;
    const StatsArgs sa{h, w, ld_h, ld_w, p.part, targets, p.target64, ignore_index, p.m, p.k, p.v,
                       static_cast<int>(word_tiles), lse, loss_rows};
    const unsigned grid = static_cast<unsigned>((m + 3) / 4);
    if (dtype == AXON_BF16) ce_stats<__nv_bfloat16><<<grid, 128, 0, s>>>(sa);
    else ce_stats<__half><<<grid, 128, 0, s>>>(sa);
    if ((rc = launch_status(what))) return rc;
  }
  if (reduction != AXON_REDUCE_NONE) {
    ce_reduce<<<1, 1024, 0, s>>>(loss_rows, targets, target_bits == 64, ignore_index, v, static_cast<int>(m),
                                 reduction == AXON_REDUCE_MEAN, loss);
    return launch_status(what);
  }
  return AXON_OK;
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
  ra.row_target = ra.row_index + g.rows;
  ra.row_lse = reinterpret_cast<float*>(ra.row_target + g.rows);
  ra.row_g = ra.row_lse + g.rows;
  ra.row_dt = ra.row_g + g.rows;
  ra.hc = ws + g.off_hc;
  const int64_t cap = 4ll * sm_count();
  ce_grad_rows<<<static_cast<unsigned>(m < cap ? m : cap), kRowThreads, 0, s>>>(ra);
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
    p.ld_dw = ld_dw;
    p.acc = reinterpret_cast<float*>(ws + g.off_acc);
    p.first = i == 0;
    p.last = i + 1 == g.pieces;
    p.band = band_of(k);
    CeParams pg = p;
    if ((rc = make_map(&p.a, ra.hc, dtype, k, g.rows, k, BK, BM, "h", what))) return rc;
    if ((rc = make_map(&p.b, wp, dtype, k, vc, ld_w, BK, BH, "w", what))) return rc;
    p.a2 = p.a;
    p.b2 = p.b;
    if ((rc = make_map(&pg.a, p.d, dtype, vc, g.rows, p.ld_d, BK, BM, "d", what))) return rc;
    if ((rc = make_map(&pg.b, wp, dtype, k, vc, ld_w, 64, BK, "w", what))) return rc;
    if ((rc = make_map(&pg.a2, p.d, dtype, vc, g.rows, p.ld_d, 64, BK, "d", what))) return rc;
    if ((rc = make_map(&pg.b2, ra.hc, dtype, k, g.rows, k, 64, BK, "h", what))) return rc;
    rc = dtype == AXON_BF16 ? run_piece<__nv_bfloat16>(p, pg, dw_dtype, g.rows, t.max_ctas, s)
                            : run_piece<__half>(p, pg, dw_dtype, g.rows, t.max_ctas, s);
    if (rc) return rc;
  }
  return AXON_OK;
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
