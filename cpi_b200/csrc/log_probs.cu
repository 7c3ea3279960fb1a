// Log probabilities of given tokens, the entropy of each row's distribution and its most probable tokens, in one pass.
//
//     m = max x,  Z = sum e^(x - m),  S = sum e^(x - m) (x - m);   log p(t) = (x_t - m) - ln Z;   H = ln Z - S / Z
//
// Sums are float32 in powers of two, a share per thread with a maximum of its own, two numbers to an instruction; sums of
// differences keep peaked rows exact.
//
// A cluster of 1 to 8 blocks of threads takes a row: each block a share of it, through 16-byte loads, four per thread in flight
// while the four before them are worked on.  The best `top`: the 32 maxima of what the threads of each lane number have met so
// far are 32 different numbers, so the top-th largest of them is a bound that the top-th best cannot be below.  It is taken
// after the first, second, fourth, ... batch, and what is not below it goes to a list in shared memory (of n numbers in random
// order a few per doubling of n: the test is one comparison per thread and batch).  Entries are 64-bit keys (value, then lowest
// index); the list is sorted by counting for each key how many are larger.  The other blocks of a cluster put their sums and
// sorted keys into the first one's shared memory and leave.  If a list runs over (a row of thousands of equal numbers) the share
// is read again, each warp keeping its best in its lanes.
// One launch, no scratch, a fixed order of sums; which key is where in the list does not matter.
// Bound by reading the logits; with few rows by the latency of a share and of joining the shares, so that then a row is shared.
//
// Numbers at the edges: -inf has probability zero (and no share in H).  A row of -inf only has no distribution: log
// probabilities -inf, entropy 0.  A row that holds NaN or +inf: log probabilities and entropy are NaN; NaN is never among the
// best.  A target below zero stands for none (0 is returned), one beyond the vocabulary gives NaN.
#include "common.cuh"
#include "f32x2.cuh"
#include "packed.cuh"

namespace cpi {
namespace lp {

constexpr int UNROLL = 4, kMaxTop = 32, kMaxWarps = 16;
constexpr int kList = 1024, kShort = 256; // keys kept beside the sums, and those of them that are sorted
constexpr int kMaxCluster = 8;
// References begin here, at a number of both types: what is below is as good as -inf unless a row has nothing else.  (As
// bfloat16 numbers are coarser, one that they would round could lie above a thread's reference, and its exponential overflow.)
constexpr float kFloor = -0x1p126f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kNone = 0x7fffffff;

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
// The exponent that a share's sums are scaled by, towards a larger reference: 0 for all that is 2^-200 or less, so that it stays
// finite where the distance is beyond float32.  Every product of it is formed: zero times NaN keeps a NaN that a share has met.
__device__ __forceinline__ float distance(float m, float top) { return fmaxf((m - top) * kLog2e, -200.f); }
struct Sums { float m, z, s; };           // largest x, sum 2^d, sum 2^d d with d = (x - m) log2 e
__device__ __forceinline__ Sums merged(Sums a, Sums b) {
  Sums t;
  t.m = fmaxf(a.m, b.m);
  const float da = distance(a.m, t.m), db = distance(b.m, t.m), fa = ex2(da), fb = ex2(db);
  // (products rounded before they are added: the same z in both lanes of a pair, so in all lanes of a warp)
  t.z = __fadd_rn(__fmul_rn(fa, a.z), __fmul_rn(fb, b.z));
  t.s = __fadd_rn(__fmul_rn(fa, fmaf(a.z, da, a.s)), __fmul_rn(fb, fmaf(b.z, db, b.s)));
  return t;
}
__device__ __forceinline__ Sums shifted(const Sums& a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.z, o), __shfl_xor_sync(0xffffffffu, a.s, o)};
}

// A number and its index as a key: larger numbers first, then lower indices.  0 is no key.
__device__ __forceinline__ int ordered(float x) {          // integers that order like the numbers
  const int b = __float_as_int(x + 0.f);                   // (-0 counts as 0)
  return b >= 0 ? b : b ^ 0x7fffffff;
}
__device__ __forceinline__ uint64_t key_of(float x, int at) {
  return ((uint64_t)((uint32_t)ordered(x) ^ 0x80000000u) << 32) | (uint32_t)~at;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const int b = (int)((uint32_t)(key >> 32) ^ 0x80000000u);
  return __int_as_float(b >= 0 ? b : b ^ 0x7fffffff);
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int src) { return __shfl_sync(0xffffffffu, (unsigned long long)v, src); }

// A warp's best keys: lane i holds the i-th, the first `top` lanes count.
struct Best {
  uint64_t k = 0, last = 0;               // this lane's; the one of lane top - 1
  __device__ __forceinline__ void offer(uint64_t key, int top) {          // every lane's key
    unsigned who = __ballot_sync(0xffffffffu, key > last);
    while (who) {
      const int src = __ffs(who) - 1;
      who &= who - 1;
      const uint64_t x = shfl64(key, src);
      if (x <= last) continue;
      const int place = __popc(__ballot_sync(0xffffffffu, k > x)), lane = threadIdx.x & 31;
      const uint64_t up = __shfl_up_sync(0xffffffffu, (unsigned long long)k, 1);
      k = lane == place ? x : lane > place ? up : k;
      last = shfl64(k, top - 1);
    }
  }
};

struct Shared {
  Sums part[kMaxWarps];
  int n_list, n_short;
  __align__(16) int lane_max[32];         // the largest that threads of each lane number have met (see ordered())
  __align__(16) int snapshot[kMaxWarps][32];      // of these, each warp's own (see bound_of())
  __align__(16) uint64_t list[kList];     // (when it has run over: every warp's best)
  __align__(16) uint64_t shorter[kShort];
  uint64_t top[kMaxTop];                  // the sorted best, 0 behind the last
  float scratch[32];
  // of the row's first block: what the cluster's blocks bring
  Sums sums[kMaxCluster];
  uint64_t tops[kMaxCluster * kMaxTop];
  unsigned long long bound;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The place of `p` in the shared memory of the cluster's block 0.
__device__ __forceinline__ uint32_t in_first(const void* p) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void put_float(uint32_t at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
__device__ __forceinline__ void put_key(uint32_t at, uint64_t v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }

// A bound for the top-th best of what the block has met: of the 32 maxima over the threads of each lane number the top-th
// largest.  Whole warps call it, with their running maxima; `together`: all of the block's, so that everyone's count.  (What some
// of the threads have met gives a bound all the same, if a lower one, and maxima only grow: no need to wait for the others.)
// The others raise the maxima meanwhile, so they are read once, into this warp's snapshot, and both the ranks and the result are
// the snapshot's: 32 different numbers that have been met, of which `top` are not below the result.  (Read a second time for the
// ranks, a maximum that has grown in between would count against its own older number, and the bound would come out too high.)
__device__ __forceinline__ float bound_of(Shared& sh, float own, int top, bool together) {
  const int lane = threadIdx.x & 31;
  const int mine = ordered(own);
  if (mine > *reinterpret_cast<volatile int*>(&sh.lane_max[lane])) atomicMax(&sh.lane_max[lane], mine);
  if (together) __syncthreads(); else __syncwarp();
  const int v = *reinterpret_cast<volatile int*>(&sh.lane_max[lane]);
  int* snapshot = sh.snapshot[threadIdx.x >> 5];
  snapshot[lane] = v;
  __syncwarp();
  int before = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int4 o = reinterpret_cast<const int4*>(snapshot)[i];
    before += (o.x > v) + (o.y > v) + (o.z > v) + (o.w > v);
  }
  // the lanes with fewer than `top` before them; the least of their numbers is the top-th largest
  const int least = __reduce_min_sync(0xffffffffu, before < top ? v : 0x7fffffff);
  return fmaxf(__int_as_float(least >= 0 ? least : least ^ 0x7fffffff), kLowest);
}

// Sorts n different keys (n <= kShort, any order, 0 behind the last up to a multiple of eight) into sh.top.  All threads call it.
__device__ __forceinline__ void sort_keys(Shared& sh, const uint64_t* keys, int n, int top) {
  for (int t = threadIdx.x; t < n; t += blockDim.x) {
    const uint64_t mine = keys[t];
    int before = 0;
    for (int i = 0; i < n; i += 8) {
      ulonglong2 o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = reinterpret_cast<const ulonglong2*>(keys + i)[u];
#pragma unroll
      for (int u = 0; u < 4; ++u) before += (o[u].x > mine) + (o[u].y > mine);
    }
    if (before < top) sh.top[before] = mine;
  }
  __syncthreads();
}
// The keys of `from` (n of them, 0 is none) that are not below `bound` go to sh.shorter; how many (more than kShort: too many).
__device__ __forceinline__ int shorten(Shared& sh, const uint64_t* from, int n, uint64_t bound) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const uint64_t k = from[i];
    if (k && k >= bound) {
      const int place = atomicAdd(&sh.n_short, 1);
      if (place < kShort) sh.shorter[place] = k;
    }
  }
  __syncthreads();
  const int have = sh.n_short;
  if (threadIdx.x < 8 && have + threadIdx.x < kShort) sh.shorter[have + threadIdx.x] = 0;
  __syncthreads();
  return have;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static constexpr uint32_t kNothing = 0xff800000u;          // -inf
  // eight numbers at a time would not fit a vector: two pairs
  static __device__ __forceinline__ float largest(const uint4& w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  // pair i of the vector, nothing below kFloor
  static __device__ __forceinline__ uint64_t get(const uint4& w, int i) {
    const float a = __uint_as_float(i ? w.z : w.x), b = __uint_as_float(i ? w.w : w.y);
    return pair(max_nan(a, kFloor), max_nan(b, kFloor));
  }
  static __device__ __forceinline__ float one(const uint4& w, int i) { return __uint_as_float(i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t kNothing = 0xff80ff80u;
  static __device__ __forceinline__ __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  static __device__ __forceinline__ float largest(const uint4& w) {
    const __nv_bfloat162 m = __hmax2(__hmax2(two(w.x), two(w.y)), __hmax2(two(w.z), two(w.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint64_t get(const uint4& w, int i) {
    const uint32_t u = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
    const __nv_bfloat162 c = __hmax2_nan(two(u), __float2bfloat162_rn(kFloor));
    const uint32_t v = *reinterpret_cast<const uint32_t*>(&c);
    return pair(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ float one(const uint4& w, int i) {
    const uint32_t u = i < 2 ? w.x : i < 4 ? w.y : i < 6 ? w.z : w.w;
    return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
  }
};

struct Params {
  const void* logits; long stride; int vocab;
  const void* targets; int n_targets, wide_targets;          // [rows, n_targets] int32, or int64
  float* logprob; float* entropy;
  float* top_v; int* top_i; int top;
  int cluster;
};

// The best of a share once more, when there were too many to list: every warp keeps its own in its lanes.
template <typename T, int NT>
__device__ __noinline__ void best_again(Shared& sh, const T* row, int head, int v0, int v1, bool ends, int vocab, int top) {
  constexpr int N = Vec<T>::N, WARPS = NT / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto key_at = [&](int at) {              // (-inf is not kept: it is filled in at the end, where there is nothing else)
    const float x = to_f32(row[at]);
    return x >= kLowest ? key_of(x, at) : 0;
  };
  Best best;
  __syncthreads();
  for (int base = v0 * N + warp * 32; base < v1 * N; base += NT) best.offer(base + lane < v1 * N ? key_at(head + base + lane) : 0, top);
  if (ends && warp == 0) {
    const int n_vec = (vocab - head) / N, rest = vocab - head - n_vec * N;
    const int at = lane < head ? lane : lane < head + rest ? vocab - rest + lane - head : kNone;
    best.offer(at == kNone ? 0 : key_at(at), top);
  }
  static_assert(kList >= WARPS * 32, "every warp's best");
  sh.list[warp * 32 + lane] = lane < top ? best.k : 0;
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < WARPS; ++w) best.offer(sh.list[w * 32 + lane], top);
    sh.top[lane] = lane < top ? best.k : 0;
  }
  __syncthreads();
}

template <typename T, bool TOP, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) log_probs_kernel(Params p) {
  __shared__ Shared sh;
  constexpr int N = Vec<T>::N, WARPS = NT / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.cluster > 1 ? (int)cluster_rank() : 0;
  const size_t r = blockIdx.x / p.cluster;
  const T* row = reinterpret_cast<const T*>(p.logits) + r * p.stride;
  // up to `head` the row is not on 16 bytes; the vectors from there on are shared out; what is left goes with the head
  const int head = min(p.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
  const int n_vec = (p.vocab - head) / N;
  const int v0 = (int)((long)n_vec * rank / p.cluster), v1 = (int)((long)n_vec * (rank + 1) / p.cluster);
  const uint4* vec = reinterpret_cast<const uint4*>(row + head);
  float m = kFloor;                        // the largest so far of this thread (not below kFloor)
  uint64_t z2 = pair(0.f, 0.f), s2 = z2;
  float bound = kLowest, own = -INFINITY;  // own: the largest of this thread, for the bound
  if (p.cluster > 1) cluster_arrive();     // (waited for before anything is put into the first block)
  if (TOP) {
    if (tid == 0) sh.n_list = sh.n_short = 0;
    if (tid < kMaxTop) { sh.top[tid] = 0; sh.lane_max[tid] = ordered(-INFINITY); }
    __syncthreads();
  }
  pdl_wait();
  pdl_launch_dependents();

  auto load = [&](uint4 (&w)[UNROLL], int base) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int at = base + u * NT;
      w[u] = at < v1 ? __ldg(vec + at) : make_uint4(Vec<T>::kNothing, Vec<T>::kNothing, Vec<T>::kNothing, Vec<T>::kNothing);
    }
  };
  uint4 next[UNROLL];
  load(next, v0 + tid);
  // the first targets' numbers, long before they are wanted
  auto target_at = [&](int i) {
    const size_t at = r * p.n_targets + i;
    return p.wide_targets ? reinterpret_cast<const long*>(p.targets)[at] : (long)reinterpret_cast<const int*>(p.targets)[at];
  };
  long target = -1;
  float target_x = 0.f;
  if (rank == 0 && tid < p.n_targets) {
    target = target_at(tid);
    if (target >= 0 && target < p.vocab) target_x = to_f32(row[target]);
  }
  auto raise = [&](float top) {
    if (top > m) {
      const float d = distance(m, top), f = ex2(d);
      s2 = mul2(fma2(z2, pair(d, d), s2), pair(f, f));
      z2 = mul2(z2, pair(f, f));
      m = top;
    }
  };
  auto add = [&](uint64_t x) {
    const uint64_t d = mul2(add2(x, pair(-m, -m)), pair(kLog2e, kLog2e));
    const float2 v = unpair(d);
    const uint64_t e = pair(ex2(v.x), ex2(v.y));
    z2 = add2(z2, e);
    s2 = fma2(e, d, s2);
  };
  auto list = [&](float x, int at) {
    const int place = atomicAdd(&sh.n_list, 1);
    if (place < kList) sh.list[place] = key_of(x, at);
  };
  if (rank == 0 && warp == 0) {            // the ends
    const int rest = p.vocab - head - n_vec * N;
    const int at = lane < head ? lane : lane < head + rest ? p.vocab - rest + lane - head : kNone;
    if (at != kNone) {
      const float x = to_f32(row[at]);
      raise(x);
      const float d = (max_nan(x, kFloor) - m) * kLog2e, e = ex2(d);
      const float2 z = unpair(z2), s = unpair(s2);
      z2 = pair(z.x + e, z.y);
      s2 = pair(fmaf(e, d, s.x), s.y);
      if (TOP && x >= kLowest) list(x, at);
    }
    __syncwarp();
  }
  const int n_batches = (v1 - v0 + NT * UNROLL - 1) / (NT * UNROLL);
  for (int b = 0; b < n_batches; ++b) {
    const int base = v0 + b * NT * UNROLL + tid;
    uint4 w[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) w[u] = next[u];
    if (b + 1 < n_batches) load(next, base + NT * UNROLL);
    float top = Vec<T>::largest(w[0]);
#pragma unroll
    for (int u = 1; u < UNROLL; ++u) top = fmaxf(top, Vec<T>::largest(w[u]));
    raise(top);
    if (TOP) own = fmaxf(own, top);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int i = 0; i < N / 2; ++i) add(Vec<T>::get(w[u], i));
    if (TOP) {
      if ((b & (b - 1)) == 0) bound = fmaxf(bound, bound_of(sh, own, p.top, b == 0));      // b = 0, 1, 2, 4, ...
      if (top >= bound) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float x = Vec<T>::one(w[u], i);
            if (x >= bound) list(x, head + (base + u * NT) * N + i);
          }
      }
    }
  }
  // ---- lanes, warps ----
  Sums a;
  {
    const float2 z = unpair(z2), s = unpair(s2);
    a = Sums{m, z.x + z.y, s.x + s.y};
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = merged(a, shifted(a, o));
  if (lane == 0) sh.part[warp] = a;
  __syncthreads();
  if (TOP) {
    const int n = sh.n_list;
    if (n <= 64) {
      if (tid < 8) sh.list[n + tid] = 0;
      __syncthreads();
      sort_keys(sh, sh.list, n, p.top);
    } else {
      int have = kShort + 1;
      if (n <= kList) have = shorten(sh, sh.list, n, key_of(fmaxf(bound, bound_of(sh, own, p.top, true)), -1));      // (index -1: below all of that value)
      if (have <= kShort) sort_keys(sh, sh.shorter, have, p.top);
      else best_again<T, NT>(sh, row, head, v0, v1, rank == 0, p.vocab, p.top);
    }
  }
  if (warp == 0) {
    a = sh.part[lane & (WARPS - 1)];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) a = merged(a, shifted(a, o));
  }
  // ---- blocks of the cluster: their sums and best go to the first one's shared memory ----
  if (p.cluster > 1) {
    cluster_wait();
    if (warp == 0) {
      if (lane == 0) {
        const uint32_t at = in_first(&sh.sums[rank]);
        put_float(at, a.m); put_float(at + 4, a.z); put_float(at + 8, a.s);
      }
      if (TOP && lane < p.top) put_key(in_first(&sh.tops[rank * p.top + lane]), sh.top[lane]);
    }
    cluster_arrive();
    if (TOP && tid == 0) { sh.bound = 0; sh.n_short = 0; }
    cluster_wait();
    if (rank != 0) return;                 // (nobody reads this block's shared memory)
    a = sh.sums[lane & (p.cluster - 1)];
    for (int o = p.cluster / 2; o > 0; o >>= 1) a = merged(a, shifted(a, o));
    if (TOP) {
      // the largest of the blocks' last ones is a bound
      const int n = p.cluster * p.top;
      if (tid < p.cluster) atomicMax(&sh.bound, (unsigned long long)sh.tops[tid * p.top + p.top - 1]);
      if (tid >= 32 && tid < 32 + kMaxTop) sh.top[tid - 32] = 0;
      __syncthreads();
      const int have = shorten(sh, sh.tops, n, sh.bound);
      sort_keys(sh, sh.shorter, have, p.top);
    }
  } else {
    if (warp == 0 && lane == 0) sh.sums[0] = a;
    __syncthreads();
    a = sh.sums[0];
  }
  bool empty = false;
  if (!(a.m > kFloor && a.m < -kFloor)) {
    // Nothing above kFloor (masks of the type's lowest value, or of -inf), or a largest number from which kFloor is further than
    // float32 goes (zero times that distance is NaN): once more, against the true maximum and the numbers as they are.
    float top = -INFINITY;
    for (int i = tid; i < p.vocab; i += NT) top = fmaxf(top, to_f32(row[i]));
    top = block_max(top, sh.scratch);
    empty = top == -INFINITY && a.z == a.z;
    float z = 0.f, s = 0.f;
    if (top > -INFINITY)
      for (int i = tid; i < p.vocab; i += NT) {
        const float x = to_f32(row[i]), d = (x - top) * kLog2e, e = ex2(d);
        z += e;
        s = e > 0.f ? fmaf(e, d, s) : s;
      }
    z = block_sum(z, sh.scratch);
    s = block_sum(s, sh.scratch);
    if (a.z == a.z) a = Sums{top, z, s};                // (else there is a NaN)
  }
  const float ln_z = logf(a.z);
  auto log_p = [&](float x) { return empty ? -INFINITY : (x - a.m) - ln_z; };
  if (tid == 0) p.entropy[r] = empty ? 0.f : ln_z - kLn2 * (a.s / a.z);
  for (int i = tid; i < p.n_targets; i += NT) {
    if (i != tid) {
      target = target_at(i);
      if (target >= 0 && target < p.vocab) target_x = to_f32(row[target]);
    }
    p.logprob[r * p.n_targets + i] = target < 0 ? 0.f : target < p.vocab ? log_p(target_x) : __int_as_float(0x7fffffff);
  }
  if (TOP && warp == 0) {
    const uint64_t key = lane < p.top ? sh.top[lane] : 0;
    float x = value_of(key);
    int at = key ? index_of(key) : kNone, have = __popc(__ballot_sync(0xffffffffu, key != 0));
    // fewer than `top` numbers above -inf: tokens of -inf follow, the lowest ids first
    for (int base = 0; have < p.top && base < p.vocab; base += 32) {
      unsigned who = __ballot_sync(0xffffffffu, base + lane < p.vocab && to_f32(row[min(base + lane, p.vocab - 1)]) == -INFINITY);
      while (who && have < p.top) {
        if (lane == have) { x = -INFINITY; at = base + __ffs(who) - 1; }
        who &= who - 1;
        ++have;
      }
    }
    if (lane < p.top) {
      p.top_v[r * p.top + lane] = at == kNone ? __int_as_float(0x7fffffff) : log_p(x);
      p.top_i[r * p.top + lane] = at == kNone ? -1 : at;
    }
  }
}

template <typename T, bool TOP, int NT>
int launch(const Params& p, int rows, cudaStream_t stream) {
  auto* kernel = log_probs_kernel<T, TOP, NT>;
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
template <typename T, bool TOP>
int launch(const Params& p, int rows, int threads, cudaStream_t stream) {
  return threads == 512 ? launch<T, TOP, 512>(p, rows, stream) : threads == 256 ? launch<T, TOP, 256>(p, rows, stream) : launch<T, TOP, 128>(p, rows, stream);
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
  while (cluster < lp::kMaxCluster && (long)rows * cluster * 2 <= enough && vocab / (cluster * 2) >= 2048) cluster *= 2;
  lp::Params p{logits, stride, vocab, targets, n_targets, wide_targets, logprob, entropy, top_v, top_i, top, cluster};
  // Threads of a block: 512 where the blocks fill no more than the device at once (8 x 202,048 float32, 64 blocks: 10.6 us, with 256 12.2).
  // More blocks than that hide each other's ends, which are many barriers long: 256 (1,000 x 151,643 bfloat16: 68 us, with 512 83, with 128
  // 75), or 128 where rows are short and many (2,000 rows of 500 / 4,000 / 16,000 float32: 9.4 / 13.9 / 29 us, with 256 16.2 / 17.6 /
  // 33; 600 of 16,000: 17.0 and 14.4).
  const int threads = (long)rows * cluster <= enough ? 512 : vocab <= 16384 && rows >= 8 * sm_count() ? 128 : 256;
  if (dtype == kF32) return top ? lp::launch<float, true>(p, rows, threads, stream) : lp::launch<float, false>(p, rows, threads, stream);
  if (dtype == kBF16) return top ? lp::launch<__nv_bfloat16, true>(p, rows, threads, stream) : lp::launch<__nv_bfloat16, false>(p, rows, threads, stream);
  set_error("log_probs: unknown dtype code %d", dtype);
  return 1;
}
CPI_PACKED(cpi_log_probs)
