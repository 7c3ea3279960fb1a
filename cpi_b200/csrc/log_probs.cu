// Log probabilities of given tokens, the entropy of each row's distribution and its most probable tokens, in one pass.
//
//     lse = m + ln Z,  m = max x,  Z = sum e^(x - m);   log p(t) = (x_t - m) - ln Z;   H = ln Z - sum e^(x - m) (x - m) / Z
//
// A cluster of 1 to 16 blocks of threads takes a row: each block a share of it, through 16-byte loads with four in flight per
// thread, every thread with a running maximum and the two sums against it in float32 (sums of differences, so that a peaked row
// loses nothing).  A warp keeps the best `top` numbers it has met in its lanes, sorted (value, then lowest index); a number
// enters when it beats the last of them and is not below the best such bound of any warp of the block.  Of n numbers in random
// order about top * ln(n / top) enter, so the test, one comparison per thread and four loads, is what it costs.  Lists and sums
// are merged warps first, then blocks over distributed shared memory: one launch, no scratch, a fixed order of sums.
// Bound by reading the logits; with few rows by the latency of a share, so that then a row is shared by 16 blocks.
//
// Numbers at the edges: -inf has probability zero (and no share in H).  A row of -inf only has no distribution: log
// probabilities -inf, entropy 0.  A row that holds NaN or +inf: log probabilities and entropy are NaN; NaN is never among the
// best.  A target below zero stands for none (0 is returned), one beyond the vocabulary gives NaN.
#include "common.cuh"

namespace cpi {
namespace lp {

constexpr int NT = 512, WARPS = NT / 32, UNROLL = 4, kMaxTop = 32;
constexpr float kFloor = -1e38f;          // running maxima begin here: what is below is as good as -inf unless a row has nothing else
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {          // the larger; NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

struct Sums { float m, z, s; };           // maximum, sum e^(x - m), sum e^(x - m) (x - m)
__device__ __forceinline__ Sums merged(Sums a, Sums b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float fa = ex2((a.m - r.m) * kLog2e), fb = ex2((b.m - r.m) * kLog2e);
  // (a factor of zero drops its side: the distance may be beyond float32)
  r.z = (fa > 0.f ? fa * a.z : 0.f) + (fb > 0.f ? fb * b.z : 0.f);
  r.s = (fa > 0.f ? fa * fmaf(a.z, a.m - r.m, a.s) : 0.f) + (fb > 0.f ? fb * fmaf(b.z, b.m - r.m, b.s) : 0.f);
  return r;
}
__device__ __forceinline__ Sums shifted(const Sums& a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.z, o), __shfl_xor_sync(0xffffffffu, a.s, o)};
}

// A warp's best numbers: lane i holds the i-th (value, index), the first `top` lanes count.
struct Best {
  float v; int i;                         // this lane's entry
  float last_v; int last_i;               // entry top - 1, in every lane
  __device__ __forceinline__ void clear() { v = last_v = -INFINITY; i = last_i = 0x7fffffff; }
  __device__ __forceinline__ bool takes(float x, int at) const { return x > last_v || (x == last_v && at < last_i); }
  __device__ __forceinline__ void put(float x, int at, int top) {          // the same (x, at) in every lane
    const bool before = v > x || (v == x && i < at);
    const int place = __popc(__ballot_sync(0xffffffffu, before)), lane = threadIdx.x & 31;
    const float uv = __shfl_up_sync(0xffffffffu, v, 1);
    const int ui = __shfl_up_sync(0xffffffffu, i, 1);
    if (lane == place) { v = x; i = at; }
    else if (lane > place) { v = uv; i = ui; }
    last_v = __shfl_sync(0xffffffffu, v, top - 1);
    last_i = __shfl_sync(0xffffffffu, i, top - 1);
  }
  // every lane's (x, at); an `at` of 0x7fffffff is never taken
  __device__ __forceinline__ void offer(float x, int at, float bound, int top) {
    unsigned who = __ballot_sync(0xffffffffu, !(x < bound) && takes(x, at));
    while (who) {
      const int src = __ffs(who) - 1;
      who &= who - 1;
      const float xv = __shfl_sync(0xffffffffu, x, src);
      const int xi = __shfl_sync(0xffffffffu, at, src);
      if (takes(xv, xi)) put(xv, xi, top);
    }
  }
};

struct Shared {
  Sums part[WARPS];
  float best_v[WARPS][kMaxTop];
  int best_i[WARPS][kMaxTop];
  // what the row's first block reads over the cluster
  Sums sums;
  float top_v[kMaxTop];
  int top_i[kMaxTop];
  float bound;
  float scratch[32];
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 32 bits of another block's shared memory at the place where `p` is in ours
__device__ __forceinline__ uint32_t peer_word(const void* p, uint32_t rank) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), v;
  asm volatile("{\n\t.reg .u32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.u32 %0, [r];\n\t}" : "=r"(v) : "r"(a), "r"(rank) : "memory");
  return v;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& w, float* x) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
  static constexpr uint32_t kNothing = 0xff800000u;          // -inf
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& w, float* x) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
  }
  static constexpr uint32_t kNothing = 0xff80ff80u;
};

struct Params {
  const void* logits; long stride; int vocab;
  const void* targets; int n_targets, wide_targets;          // [rows, n_targets] int32, or int64
  float* logprob; float* entropy;
  float* top_v; int* top_i; int top;
  int cluster;
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(NT) log_probs_kernel(Params p) {
  __shared__ Shared sh;
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.cluster > 1 ? (int)cluster_rank() : 0;
  const size_t r = blockIdx.x / p.cluster;
  const T* row = reinterpret_cast<const T*>(p.logits) + r * p.stride;
  // up to `head` the row is not on 16 bytes; the vectors from there on are shared out; what is left goes with the head
  const int head = min(p.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
  const int n_vec = (p.vocab - head) / N;
  const int v0 = (int)((long)n_vec * rank / p.cluster), v1 = (int)((long)n_vec * (rank + 1) / p.cluster);
  const uint4* vec = reinterpret_cast<const uint4*>(row + head);
  Sums a{kFloor, 0.f, 0.f};
  Best best;
  best.clear();
  if (TOP && tid == 0) sh.bound = -INFINITY;
  if (TOP) __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  auto add = [&](const float* x, int n) {
    float top = x[0];
    for (int i = 1; i < n; ++i) top = fmaxf(top, x[i]);
    if (top > a.m) {
      const float f = ex2((a.m - top) * kLog2e);
      a.s = f > 0.f ? f * fmaf(a.z, a.m - top, a.s) : 0.f;
      a.z *= f;
      a.m = top;
    }
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float d = max_nan(x[i], kFloor) - a.m, e = ex2(d * kLog2e);
      a.z += e;
      a.s = fmaf(e, d, a.s);
    }
    return top;
  };
  if (rank == 0 && warp == 0) {            // the ends
    const int rest = p.vocab - head - n_vec * N;
    const int at = lane < head ? lane : lane < head + rest ? p.vocab - rest + lane - head : 0x7fffffff;
    float x[1] = {at == 0x7fffffff ? -INFINITY : to_f32(row[at])};
    if (at != 0x7fffffff) add(x, 1);
    __syncwarp();
    if (TOP) best.offer(x[0], at, -INFINITY, p.top);
  }
  for (int base = v0 + warp * 32; base < v1; base += NT * UNROLL) {
    uint4 w[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int at = base + u * NT + lane;
      w[u] = at < v1 ? __ldg(vec + at) : make_uint4(Vec<T>::kNothing, Vec<T>::kNothing, Vec<T>::kNothing, Vec<T>::kNothing);
    }
    float x[UNROLL * N];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) Vec<T>::get(w[u], x + u * N);
    const float top = add(x, UNROLL * N);
    if (TOP) {
      const float bound = *reinterpret_cast<volatile float*>(&sh.bound);
      if (__any_sync(0xffffffffu, top >= bound && top >= best.last_v)) {
        // rare: the numbers are read once more, one place of every lane's vectors at a time
#pragma unroll 1
        for (int u = 0; u < UNROLL; ++u) {
          const int at = base + u * NT + lane;
#pragma unroll 1
          for (int i = 0; i < N; ++i) {
            const int index = head + at * N + i;
            best.offer(at < v1 ? to_f32(row[index]) : -INFINITY, at < v1 ? index : 0x7fffffff, bound, p.top);
          }
        }
        // (a plain store: whichever of two warps comes last, the number is a bound)
        if (lane == 0 && best.last_v > bound) *reinterpret_cast<volatile float*>(&sh.bound) = best.last_v;
      }
    }
  }
  // ---- lanes, warps ----
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = merged(a, shifted(a, o));
  if (lane == 0) sh.part[warp] = a;
  if (TOP) { sh.best_v[warp][lane] = best.v; sh.best_i[warp][lane] = best.i; }
  __syncthreads();
  if (warp == 0) {
    a = sh.part[0];
    for (int w = 1; w < WARPS; ++w) {
      a = merged(a, sh.part[w]);
      if (TOP) best.offer(sh.best_v[w][lane], lane < p.top ? sh.best_i[w][lane] : 0x7fffffff, -INFINITY, p.top);
    }
    if (lane == 0) sh.sums = a;
    if (TOP) { sh.top_v[lane] = best.v; sh.top_i[lane] = best.i; }
  }
  // ---- blocks of the cluster ----
  if (p.cluster > 1) {
    cluster_sync();
    if (rank == 0 && warp == 0) {
      for (int c = 1; c < p.cluster; ++c) {
        const Sums b{__uint_as_float(peer_word(&sh.sums.m, c)), __uint_as_float(peer_word(&sh.sums.z, c)), __uint_as_float(peer_word(&sh.sums.s, c))};
        a = merged(a, b);
        if (TOP) {
          const float x = __uint_as_float(peer_word(&sh.top_v[lane], c));
          const int at = (int)peer_word(&sh.top_i[lane], c);
          best.offer(x, lane < p.top ? at : 0x7fffffff, -INFINITY, p.top);
        }
      }
      if (lane == 0) sh.sums = a;
    }
    cluster_sync();                        // nobody leaves while its shared memory is read
  }
  if (rank != 0) return;
  __syncthreads();
  a = sh.sums;
  bool empty = false;
  if (a.m <= kFloor) {
    // nothing above -1e38 (masks of the type's lowest value, or of -inf): once more, against the true maximum
    float top = -INFINITY;
    for (int i = tid; i < p.vocab; i += NT) top = fmaxf(top, to_f32(row[i]));
    top = block_max(top, sh.scratch);
    empty = top == -INFINITY && a.z == a.z;
    float z = 0.f, s = 0.f;
    if (top > -INFINITY)
      for (int i = tid; i < p.vocab; i += NT) {
        const float x = to_f32(row[i]), d = x - top, e = ex2(d * kLog2e);
        z += e;
        s = e > 0.f ? fmaf(e, d, s) : s;
      }
    z = block_sum(z, sh.scratch);
    s = block_sum(s, sh.scratch);
    if (a.z == a.z) a = Sums{top, z, s};   // (else there is a NaN)
  }
  const float ln_z = logf(a.z);
  auto log_p = [&](float x) { return empty ? -INFINITY : (x - a.m) - ln_z; };
  if (tid == 0) p.entropy[r] = empty ? 0.f : ln_z - a.s / a.z;
  for (int i = tid; i < p.n_targets; i += NT) {
    const size_t at = r * p.n_targets + i;
    const long t = p.wide_targets ? reinterpret_cast<const long*>(p.targets)[at] : (long)reinterpret_cast<const int*>(p.targets)[at];
    p.logprob[at] = t < 0 ? 0.f : t < p.vocab ? log_p(to_f32(row[t])) : __int_as_float(0x7fffffff);
  }
  if (TOP && warp == 0 && lane < p.top) {
    const bool none = best.i == 0x7fffffff;                  // fewer numbers than that: the others are NaN
    p.top_v[r * p.top + lane] = none ? __int_as_float(0x7fffffff) : log_p(best.v);
    p.top_i[r * p.top + lane] = none ? -1 : best.i;
  }
}

template <typename T, bool TOP>
int launch(const Params& p, int rows, cudaStream_t stream) {
  auto* kernel = log_probs_kernel<T, TOP>;
  if (p.cluster > 8) {
    static bool ready[64] = {};            // per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || !ready[dev]) {
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      cudaGetLastError();
      if (dev >= 0 && dev < 64) ready[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * p.cluster);
  cfg.blockDim = dim3(NT);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  count_launch();
  cudaLaunchKernelEx(&cfg, kernel, p);
  return check_launch("log_probs");
}

}  // namespace lp
}  // namespace cpi

using namespace cpi;

extern "C" int cpi_log_probs_max_top() { return lp::kMaxTop; }

// logits [rows, vocab] float32 or bfloat16, `stride` elements between rows; targets [rows, n_targets] int32, or int64 with
// `wide_targets`; logprob [rows, n_targets], entropy [rows], top_v and top_i [rows, top] (top 0: none).
extern "C" int cpi_log_probs(const void* logits, int dtype, long stride, int rows, int vocab, const void* targets, int n_targets,
                             int wide_targets, float* logprob, float* entropy, float* top_v, int* top_i, int top, cudaStream_t stream) {
  if (rows == 0) return 0;
  CPI_REQUIRE(vocab >= 1 && rows >= 0 && rows <= (1 << 26), "log_probs: %d rows of %d", rows, vocab);
  CPI_REQUIRE(top >= 0 && top <= lp::kMaxTop && top <= vocab, "log_probs: the best %d of %d (at most %d)", top, vocab, lp::kMaxTop);
  // Rows alone fill the device from two blocks of threads per SM on; below, a row is shared by as many as keep 2,048 numbers each.
  int cluster = 1;
  const long enough = 2l * sm_count();
  while (cluster < 16 && (long)rows * cluster * 2 <= enough && vocab / (cluster * 2) >= 2048) cluster *= 2;
  lp::Params p{logits, stride, vocab, targets, n_targets, wide_targets, logprob, entropy, top_v, top_i, top, cluster};
  if (dtype == kF32) return top ? lp::launch<float, true>(p, rows, stream) : lp::launch<float, false>(p, rows, stream);
  if (dtype == kBF16) return top ? lp::launch<__nv_bfloat16, true>(p, rows, stream) : lp::launch<__nv_bfloat16, false>(p, rows, stream);
  set_error("log_probs: unknown dtype code %d", dtype);
  return 1;
}
