// Global gradient norm over a list of tensors, and clipping.
//
//   norm = sqrt(sum over tensors and elements of x^2)
//   scale = min(1, max_norm / (norm + eps));  y = scale * x
//
// The list's tensors are cut into chunks of 32 KB (a chunk never straddles two
// tensors), numbered through the list and dealt in turn to the CTAs of a
// persistent grid: every CTA carries the same bytes whatever the tensors'
// sizes, and the CTAs move through memory side by side. The tensor table
// travels as a kernel argument (no copy to the device, nothing to keep
// between calls; a captured graph holds it), so a list longer than the table
// takes several launches.
//
// Norm: each thread squares and adds 128 bytes of a chunk in fp32 (chains of a
// few elements), then adds that to a float64 running sum; the CTA's float64
// partial goes to its own workspace slot, and the slots are added in a fixed
// order by whoever needs the total: no atomics, the same bits every time.
// HBM-bound: one read of the gradients. 0.87e9 bf16 gradients: 253-267 us,
// 6.5-6.9 TB/s, 1.0-1.05 of a copy's rate (contiguous ranges took 2% longer, 16 KB
// chunks 14%).
//
// Clip: the norm kernel, then a kernel whose CTAs each add up the slots (a few
// KB, from L2) and scale their chunks, last ones first: what the first kernel
// read last is still in L2. The same gradients: 857-871 us, in place or not, of
// which three passes at the copy rate are 800.
#include "common.cuh"

namespace axon {
namespace {

constexpr int kThreads = 256;
constexpr int kChunkBytes = 32768;
constexpr int kVecs = kChunkBytes / 16 / kThreads;  // 16-byte packets a thread takes of a chunk
constexpr int kCtasPerSm = 4;

// One launch's share of the list. `first[i]` is tensor i's first chunk within
// this launch; first[count] the launch's chunk count.
template <int CAP>
struct GradTable {
  const void* in[CAP];
  void* out[CAP];
  int64_t n[CAP];
  uint32_t first[CAP + 1];
  uint8_t dtype[CAP];
  int32_t count;
};

// Sum of v over the CTA in a fixed order, returned to every thread.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double warp_part[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) s += warp_part[i];
  __syncthreads();
  return s;
}

// A chunk as bytes: a head up to the first 16-byte boundary, whole packets,
// a tail. Loads and stores are the same for every element type; only the
// arithmetic on a packet looks at it.
struct Chunk {
  const char* p;
  int bytes, head, vecs;
};

__device__ __forceinline__ Chunk chunk_of(const void* base, int64_t numel, int dt, int64_t local) {
  const int64_t all = numel * (dt == AXON_F32 ? 4 : 2);
  Chunk c;
  c.p = static_cast<const char*>(base) + local * kChunkBytes;
  const int64_t left = all - local * kChunkBytes;
  c.bytes = left < kChunkBytes ? static_cast<int>(left) : kChunkBytes;
  const int to_boundary = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(c.p) & 15u)) & 15u);
  c.head = to_boundary < c.bytes ? to_boundary : c.bytes;
  c.vecs = (c.bytes - c.head) >> 4;
  return c;
}

// Element j of the head and tail elements of a chunk (fewer than 16 in all),
// as a byte offset into the chunk, or -1.
__device__ __forceinline__ int edge_offset(const Chunk& c, int es, int j) {
  const int heads = c.head / es;
  if (j < heads) return j * es;
  const int off = c.head + c.vecs * 16 + (j - heads) * es;
  return off < c.bytes ? off : -1;
}

// The squares of a packet's elements, added to two sums of 32-bit lanes.
__device__ __forceinline__ void packet_squares(uint4 u, int dt, float* acc) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dt == AXON_F32) {
      const float x = __uint_as_float(w[i]);
      acc[i] = fmaf(x, x, acc[i]);
    } else {
      float lo, hi;
      if (dt == AXON_BF16) {
        lo = __uint_as_float(w[i] << 16);
        hi = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        lo = f.x;
        hi = f.y;
      }
      acc[i] = fmaf(lo, lo, fmaf(hi, hi, acc[i]));
    }
  }
}

// This thread's sum of squares of a chunk.
__device__ __forceinline__ float chunk_squares(const Chunk& c, int dt) {
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const uint4* body = reinterpret_cast<const uint4*>(c.p + c.head);
  uint4 v[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int at = i * kThreads + threadIdx.x;
    v[i] = at < c.vecs ? body[at] : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < kVecs; ++i) packet_squares(v[i], dt, acc);
  if (threadIdx.x < 16) {
    const int es = dt == AXON_F32 ? 4 : 2;
    const int off = edge_offset(c, es, threadIdx.x);
    if (off >= 0) {
      const float x = load_any(c.p + off, 0, dt);
      acc[0] = fmaf(x, x, acc[0]);
    }
  }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

template <int CAP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    grad_squares(const __grid_constant__ GradTable<CAP> t, double* __restrict__ part) {
  const uint32_t chunks = t.first[t.count];
  pdl_wait();
  double sum = 0.0;
  int i = 0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    while (c >= t.first[i + 1]) ++i;
    const int dt = t.dtype[i];
    sum += static_cast<double>(chunk_squares(chunk_of(t.in[i], t.n[i], dt, c - t.first[i]), dt));
  }
  pdl_trigger();
  sum = block_sum(sum);
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

struct ClipArgs {
  const double* part;
  int parts;
  float max_norm, eps;
  float* norm;
  float* scale;
};

// min(1, max_norm / (norm + eps)); a NaN norm gives a NaN scale, and gradients
// that are all zero with eps = 0 are left as they are.
__device__ __forceinline__ float clip_scale(float norm, float max_norm, float eps) {
  const float d = norm + eps;
  if (d == 0.f) return 1.f;
  const float c = max_norm / d;
  return c > 1.f ? 1.f : c;
}

__device__ __forceinline__ float total_norm(const double* part, int parts) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) s += __ldcg(part + i);
  return static_cast<float>(sqrt(block_sum(s)));
}

__global__ void __launch_bounds__(kThreads) grad_norm_finish(ClipArgs a) {
  pdl_wait();
  const float norm = total_norm(a.part, a.parts);
  if (threadIdx.x == 0) {
    if (a.norm) *a.norm = norm;
    if (a.scale) *a.scale = clip_scale(norm, a.max_norm, a.eps);
  }
}

__device__ __forceinline__ uint4 scale_packet(uint4 u, int dt, float scale) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dt == AXON_F32) {
      w[i] = __float_as_uint(__uint_as_float(w[i]) * scale);
    } else if (dt == AXON_BF16) {
      const __nv_bfloat162 r = __floats2bfloat162_rn(__uint_as_float(w[i] << 16) * scale,
                                                     __uint_as_float(w[i] & 0xffff0000u) * scale);
      w[i] = *reinterpret_cast<const uint32_t*>(&r);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      const __half2 r = __floats2half2_rn(f.x * scale, f.y * scale);
      w[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void scale_one(const void* p, void* q, int dt, float scale) {
  const float x = load_any(p, 0, dt) * scale;
  if (dt == AXON_F32) *static_cast<float*>(q) = x;
  else if (dt == AXON_BF16) *static_cast<__nv_bfloat16*>(q) = __float2bfloat16_rn(x);
  else *static_cast<__half*>(q) = __float2half_rn(x);
}

// STREAM: reads and writes that leave L2 alone (see run_lists).
template <bool STREAM>
__device__ __forceinline__ void scale_chunk(const Chunk& c, char* q, int dt, float scale) {
  const int es = dt == AXON_F32 ? 4 : 2;
  if (((reinterpret_cast<uintptr_t>(c.p) ^ reinterpret_cast<uintptr_t>(q)) & 15u) != 0) {
    // input and output start at different places of a 16-byte packet
    for (int off = threadIdx.x * es; off < c.bytes; off += kThreads * es) scale_one(c.p + off, q + off, dt, scale);
    return;
  }
  const uint4* src = reinterpret_cast<const uint4*>(c.p + c.head);
  uint4* dst = reinterpret_cast<uint4*>(q + c.head);
  uint4 v[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int at = i * kThreads + threadIdx.x;
    v[i] = at < c.vecs ? (STREAM ? __ldcs(src + at) : src[at]) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int at = i * kThreads + threadIdx.x;
    if (at >= c.vecs) continue;
    const uint4 r = scale_packet(v[i], dt, scale);
    if (STREAM) __stcs(dst + at, r);
    else dst[at] = r;
  }
  if (threadIdx.x < 16) {
    const int off = edge_offset(c, es, threadIdx.x);
    if (off >= 0) scale_one(c.p + off, q + off, dt, scale);
  }
}

template <int CAP, bool STREAM>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    grad_scale(const __grid_constant__ GradTable<CAP> t, ClipArgs a) {
  const uint32_t chunks = t.first[t.count];
  pdl_wait();
  const float norm = total_norm(a.part, a.parts);
  const float scale = clip_scale(norm, a.max_norm, a.eps);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (a.norm) *a.norm = norm;
    if (a.scale) *a.scale = scale;
  }
  int i = t.count - 1;
  for (int64_t at = (static_cast<int64_t>(chunks) - 1 - blockIdx.x) / gridDim.x; at >= 0 && blockIdx.x < chunks; --at) {
    const uint32_t c = static_cast<uint32_t>(at) * gridDim.x + blockIdx.x;
    while (c < t.first[i]) --i;
    if (scale == 1.f && t.in[i] == t.out[i]) continue;  // in place and nothing to clip
    const int dt = t.dtype[i];
    const int64_t local = c - t.first[i];
    scale_chunk<STREAM>(chunk_of(t.in[i], t.n[i], dt, local), static_cast<char*>(t.out[i]) + local * kChunkBytes, dt, scale);
  }
}

// ---- host side -------------------------------------------------------------------

constexpr int kSmallTable = 24;   // ~0.7 KB of arguments
constexpr int kLargeTable = 512;  // ~14.5 KB (the limit is 32764 bytes)

struct GradLists {
  const void* const* in;
  void* const* out;
  const int64_t* n;
  const int32_t* dtype;
  int64_t count;
};

int64_t chunks_of(int64_t n, int32_t dtype) {
  const int64_t per = kChunkBytes / dtype_size(dtype);
  return (n + per - 1) / per;
}

int check_lists(const char* what, const GradLists& g) {
  if (g.count < 0) return fail(AXON_E_SHAPE, "%s: negative tensor count", what);
  if (g.count > 0 && (!g.in || !g.n || !g.dtype)) return fail(AXON_E_ARG, "%s: NULL list", what);
  uint64_t chunks = 0;
  for (int64_t i = 0; i < g.count; ++i) {
    if (!valid_dtype(g.dtype[i]))
      return fail(AXON_E_UNSUPPORTED, "%s: tensor %lld: unsupported dtype %d", what, (long long)i, g.dtype[i]);
    if (g.n[i] < 0 || g.n[i] > (int64_t{1} << 44))
      return fail(AXON_E_SHAPE, "%s: tensor %lld: size out of range", what, (long long)i);
    if (g.n[i] > 0 && (!g.in[i] || (g.out && !g.out[i])))
      return fail(AXON_E_ARG, "%s: tensor %lld: NULL pointer", what, (long long)i);
    const uintptr_t es = dtype_size(g.dtype[i]);
    if (reinterpret_cast<uintptr_t>(g.in[i]) % es || (g.out && reinterpret_cast<uintptr_t>(g.out[i]) % es))
      return fail(AXON_E_ALIGN, "%s: tensor %lld: pointer not aligned to its element", what, (long long)i);
    chunks += static_cast<uint64_t>(chunks_of(g.n[i], g.dtype[i]));
  }
  if (chunks > 0x7fffffffull) return fail(AXON_E_SHAPE, "%s: more than 32 TB of gradients", what);
  return AXON_OK;
}

int64_t launches_of(int64_t count) { return count <= kSmallTable ? 1 : (count + kLargeTable - 1) / kLargeTable; }

// Workspace slots of a list: one per CTA of each launch.
int64_t slots_of(int64_t count) { return launches_of(count) * sm_count() * kCtasPerSm; }

template <int CAP, typename F>
int for_each_table(const GradLists& g, F&& f) {
  int64_t i = 0;
  do {
    GradTable<CAP> t{};
    uint32_t chunks = 0;
    while (i < g.count && t.count < CAP) {
      if (g.n[i] > 0) {
        t.in[t.count] = g.in[i];
        t.out[t.count] = g.out ? g.out[i] : nullptr;
        t.n[t.count] = g.n[i];
        t.first[t.count] = chunks;
        t.dtype[t.count] = static_cast<uint8_t>(g.dtype[i]);
        chunks += static_cast<uint32_t>(chunks_of(g.n[i], g.dtype[i]));
        ++t.count;
      }
      ++i;
    }
    for (int j = t.count; j <= CAP; ++j) t.first[j] = chunks;
    const int64_t cap = static_cast<int64_t>(sm_count()) * kCtasPerSm;
    const int grid = static_cast<int>(chunks < cap ? (chunks ? chunks : 1) : cap);
    int rc = f(t, grid);
    if (rc) return rc;
  } while (i < g.count);
  return AXON_OK;
}

template <int CAP>
int run_lists(const char* what, const GradLists& g, ClipArgs a, double* part, cudaStream_t s) {
  int slots = 0;
  int rc = for_each_table<CAP>(g, [&](const GradTable<CAP>& t, int grid) {
    launch_k(grad_squares<CAP>, dim3(grid), dim3(kThreads), 0, s, t, part + slots);
    slots += grid;
    return launch_status(what);
  });
  if (rc) return rc;
  a.part = part;
  a.parts = slots;
  if (!g.out) {
    launch_k(grad_norm_finish, dim3(1), dim3(kThreads), 0, s, a);
    return launch_status(what);
  }
  // Gradients that fit L2 (126 MB) are still there for the second pass if its
  // writes do not push them out: streaming (66 MB: 7% less time than without). Of
  // more than that little is left, and plain accesses are faster (0.8 GB: 2.5%
  // less).
  int64_t bytes = 0;
  for (int64_t i = 0; i < g.count; ++i) bytes += g.n[i] * dtype_size(g.dtype[i]);
  const bool stream = bytes < (126ll << 20);
  return for_each_table<CAP>(g, [&](const GradTable<CAP>& t, int grid) {
    if (stream) launch_k(grad_scale<CAP, true>, dim3(grid), dim3(kThreads), 0, s, t, a);
    else launch_k(grad_scale<CAP, false>, dim3(grid), dim3(kThreads), 0, s, t, a);
    return launch_status(what);
  });
}

int run(const char* what, const GradLists& g, const ClipArgs& a, void* workspace, int64_t workspace_bytes,
        void* stream) {
  int rc = check_lists(what, g);
  if (rc) return rc;
  if (!(a.max_norm >= 0.f)) return fail(AXON_E_ARG, "%s: max_norm must be >= 0", what);
  if (!(a.eps >= 0.f)) return fail(AXON_E_ARG, "%s: eps must be >= 0", what);
  const int64_t need = slots_of(g.count) * 8;
  if (!workspace || workspace_bytes < need)
    return fail(AXON_E_ARG, "%s: workspace of %lld bytes needed", what, (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) & 7u) return fail(AXON_E_ALIGN, "%s: workspace must be 8-byte aligned", what);
  double* part = static_cast<double*>(workspace);
  return g.count <= kSmallTable ? run_lists<kSmallTable>(what, g, a, part, as_stream(stream))
                                : run_lists<kLargeTable>(what, g, a, part, as_stream(stream));
}

}  // namespace
}  // namespace axon

using namespace axon;

extern "C" {

int64_t axon_grad_norm_workspace_bytes(int64_t count) {
  if (count < 0) return fail(AXON_E_SHAPE, "axon_grad_norm: negative tensor count");
  return slots_of(count) * 8;
}

int axon_grad_norm(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int64_t count, float max_norm,
                   float eps, float* norm, float* scale, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!norm && !scale) return fail(AXON_E_ARG, "axon_grad_norm: norm and scale are both NULL");
  GradLists g{grads, nullptr, sizes, dtypes, count};
  return run("axon_grad_norm", g, ClipArgs{nullptr, 0, max_norm, eps, norm, scale}, workspace, workspace_bytes, stream);
}

int axon_clip_grads(const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* dtypes,
                    int64_t count, float max_norm, float eps, float* norm, void* workspace, int64_t workspace_bytes,
                    void* stream) {
  if (count > 0 && !outs) return fail(AXON_E_ARG, "axon_clip_grads: NULL list");
  GradLists g{grads, outs, sizes, dtypes, count};
  if (!outs) {
    static void* const none[1] = {nullptr};
    g.out = none;
  }
  return run("axon_clip_grads", g, ClipArgs{nullptr, 0, max_norm, eps, norm, nullptr}, workspace, workspace_bytes, stream);
}

}  // extern "C"
