// Decode attention over the cache in 8 bits (kv8.cuh): one new token per sequence, its own block of 64 positions in bfloat16 (the
// sequence's tail), the complete blocks before it as codes with a scale per block and head.
//
// A block of threads serves one (split, key/value head, token).  Its warps take half pages in turn (a tile: 32 positions x D bytes)
// and stream them through shared-memory slots of their own: keys, values, keys, ... (TMA boxes of 128 bytes with the 128-byte
// swizzle), the next one asked for as soon as a slot has been read.  A slot's rounds are waited for by one warp, in order: a
// wait for a parity may be one round behind and no more.  Every warp runs an online softmax of its own:
//     S^T = K Q^T     m16n8k16 with the positions as M (two tiles of 16) and the group's heads as N (8,
//                     or twice 8): with heads as M half of the rows would be empty in the usual groups of 4 to 8, and a lane
//                     then holds the maxima of the heads that its outputs belong to.  The codes become float16 in registers: an int8
//                     c as 1024 + (c + 128) by putting its byte under the exponent of 1024, less 1152; e4m3 by the hardware's
//                     conversion; both exact.  Which positions of k a lane's bytes fill is free as long as Q's do the same, so four
//                     neighbouring bytes of a row need no shuffle.
//     O^T += V^T P^T  values by transposing loads: a pair of bytes is a pair of features, even features form the upper half of
//                     M, odd ones the lower.  P^T comes out of S^T's registers by movmatrix.
// What a warp does for a tile is one long chain of dependent steps, so the count of warps decides: 64 sequences of up to 16,384
// positions (40/8 heads of 128, e4m3) took 204 us with eight warps an SM at a page each (3,400 cycles a page, the data long there).
// The queries are float16 too, each head's divided by a power of two that brings its largest element to 2^14 (11 bits of
// significand hold bfloat16's 8 exactly; float16's smallest step is 2^-24, so an element loses bits only from 2^-31 of the
// largest on; products stay below 2^24, far from float32's ends).  Scales act on scores in float32; the value scale 2^e enters
// the exponent: a probability is p = 2^(s + e - m) with m the maximum of s + e, and the sum takes p 2^-e.  So blocks of any scale
// share one accumulator, at no operation per output.
// p is rounded to float16 (11 bits) against a reference m that is raised when s + e has outgrown it by 2^8, so the largest p lies
// between 2^6 and 2^14: what is 2^-20 of the largest still has all its bits, smaller terms are off by 2^-31 of the largest at most.
// (bfloat16 would keep 8 bits of all of them, but codes cost twice as many operations to become bfloat16.)  Sums, maxima and
// outputs are float32.
//
// The tail: four warps take 16 positions each in bfloat16, straight from memory (one page at most, in the last split); its p is
// bfloat16 like the values that it is multiplied by (outputs are off by 0.0016 to 0.0018, what rounding them takes is 0.0016).  A token
// that completes its block (position 63 of 64) has its tail turned into codes, for the steps after this one, by the last split.
// Rows of masked positions are zeros before they are multiplied: what an earlier sequence left cannot reach a result.
// Waits are bounded as in attention_decode.cu.
#include "kv8.cuh"
#include "packed.cuh"
#include <cuda.h>

namespace cpi {
namespace tc {
int get_map_2d_bf16(const void* ptr, uint64_t inner, uint64_t rows, uint64_t row_stride_bytes, uint32_t box_inner,
                    uint32_t box_rows, CUtensorMap* out);
}
namespace dec8 {

using kv8::PAGE;
constexpr uint32_t kSpinLimit = 1u << 24;
constexpr float kSlack = 8.f, kLift = 6.f;        // p = 2^(s + e - m + kLift), m raised when s + e exceeds it by kSlack
constexpr int kTailUnits = 2;                     // a tail's bytes, in pages of codes
constexpr int kMaxSplits = 256;
constexpr int kMaxCluster = 8;                    // splits that are joined over distributed shared memory

struct Params {
  const __nv_bfloat16* q; __nv_bfloat16* out;     // [T, NH, D]
  const float *k_scale, *v_scale;                 // [n_pages, NKV]
  const __nv_bfloat16 *k_tail, *v_tail;           // [n_slots, NKV, 64, D]
  uint8_t *k, *v; float *k_scale_w, *v_scale_w;   // what a completed block is written to
  const int* page_table; int max_blocks, n_pages, n_slots, n_seqs;
  const int *token_seq, *token_pos, *seq_slot;
  int n_heads, n_kv_heads;
  int window_kind, window_size, keep_first;
  float scale_log2, cap_in, cap_out;              // soft cap c > 0: scale / c and c log2(e); else 0
  int n_splits;
  bool clustered;                                 // the splits of a (token, key/value head) are a cluster
  float* part_o; float2* part_ml;                 // [T, NH, splits, D], [T, NH, splits]
  const float* sink;
  int* error_flag;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
// false when the wait ran out here or in another warp
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* aborted) {
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 255u && *aborted) return false;
  }
  *aborted = 1;
  return false;
}
__device__ __forceinline__ void tma_load_2d(void* smem, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(smem_u32(smem)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t s) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t s) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ int window_low(int kind, int size, int pos) {
  if (kind == 1) return (pos / size) * size;
  if (kind == 2) return max(0, pos - size + 1);
  return 0;
}
// 2^(sink - m), in the units of p; a sink far above every score gives a huge finite sum
__device__ __forceinline__ float sink_term(const float* sink, int head, float m) {
  return sink ? exp2f(fminf(sink[head] * 1.4426950408889634f - m + kLift, 120.f)) : 0.f;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Two floats at the place of `at` (an address in this block's shared memory) in block `rank` of the cluster.
__device__ __forceinline__ float2 peer_pair(uint32_t at, uint32_t rank) {
  float2 v;
  asm volatile("{\n\t.reg .u32 r;\n\tmapa.shared::cluster.u32 r, %2, %3;\n\tld.shared::cluster.v2.f32 {%0, %1}, [r];\n\t}"
               : "=f"(v.x), "=f"(v.y) : "r"(at), "r"(rank) : "memory");
  return v;
}
// The four codes of a word as two pairs of float16: bytes (0, 1) and (2, 3), or with SPLIT bytes (0, 2) and (1, 3).
template <int FMT, bool SPLIT> __device__ __forceinline__ void numbers(uint32_t w, uint32_t& a, uint32_t& b) {
  if (FMT == kv8::kInt8) {
    w ^= 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));              // 1024 + 128
    uint32_t x = __byte_perm(w, 0x64646464u, SPLIT ? 0x4240 : 0x4140), y = __byte_perm(w, 0x64646464u, SPLIT ? 0x4341 : 0x4342);
    __half2 u = __hsub2(*reinterpret_cast<__half2*>(&x), off), v = __hsub2(*reinterpret_cast<__half2*>(&y), off);
    a = *reinterpret_cast<uint32_t*>(&u);
    b = *reinterpret_cast<uint32_t*>(&v);
  } else {
    if (SPLIT) w = __byte_perm(w, 0u, 0x3120);
    a = kv8::e4m3x2_f16x2((uint16_t)w);
    b = kv8::e4m3x2_f16x2((uint16_t)(w >> 16));
  }
}

template <int D, int HT> struct Shape {
  static constexpr int WARPS = HT == 1 ? 8 : 4;             // (with two tiles of heads a thread needs twice the registers)
  static constexpr int NT = WARPS * 32;
  static constexpr int POS = 32;                            // positions of a tile
  static constexpr int TILE = POS * D;                      // bytes of it
  static constexpr int LINES = TILE / 128;                  // the tile as lines of 128 bytes (one, or half, a position each)
  static constexpr int SLOTS = (D == 128 ? 3 : 6) * (HT == 1 ? 1 : 2);       // tiles of keys or values that a warp has on their way or reads
  static constexpr int RING = WARPS * SLOTS * TILE;
  static constexpr int MERGE = WARPS * HT * 8 * D * 4;
  static constexpr int SMEM = (RING > MERGE ? RING : MERGE) + 1024;
};
// Byte offset of the 16-byte chunk `c` of position `row` in a tile, as the copy engine's 128-byte swizzle leaves it.
template <int D> __device__ __forceinline__ uint32_t chunk_at(int row, int c) {
  const int at = row * (D / 16) + c, line = at >> 3;
  return (uint32_t)(line * 128 + (((at & 7) ^ (line & 7)) << 4));
}

// A block of threads turns a token's tails [64, D] into codes and scales, for keys and values.
template <int D, int FMT, int NT>
__device__ __forceinline__ void hold_tail(const __nv_bfloat16* k_tail, const __nv_bfloat16* v_tail, uint8_t* k_to, uint8_t* v_to, float* k_scale,
                                          float* v_scale, uint32_t* top_s) {
  constexpr int PER = PAGE * D / 8 / NT;
  const int tid = threadIdx.x;
  const uint4 *ks = reinterpret_cast<const uint4*>(k_tail), *vs = reinterpret_cast<const uint4*>(v_tail);
  uint4 k[PER], v[PER];
  uint32_t tk = 0, tv = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) { k[i] = ks[tid + i * NT]; v[i] = vs[tid + i * NT]; }
#pragma unroll
  for (int i = 0; i < PER; ++i) { tk = max(tk, kv8::top_of(k[i])); tv = max(tv, kv8::top_of(v[i])); }
  tk = __reduce_max_sync(0xffffffffu, tk);
  tv = __reduce_max_sync(0xffffffffu, tv);
  if ((tid & 31) == 0) { top_s[tid >> 5] = tk; top_s[8 + (tid >> 5)] = tv; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) { tk = max(tk, top_s[w]); tv = max(tv, top_s[8 + w]); }
  const int ek = kv8::scale_exponent<FMT>(__uint_as_float(tk << 16)), ev = kv8::scale_exponent<FMT>(__uint_as_float(tv << 16));
  const float ik = kv8::power_of_two(-ek), iv = kv8::power_of_two(-ev);
  uint2 *kd = reinterpret_cast<uint2*>(k_to), *vd = reinterpret_cast<uint2*>(v_to);
#pragma unroll
  for (int i = 0; i < PER; ++i) { kd[tid + i * NT] = kv8::codes8<FMT>(k[i], ik); vd[tid + i * NT] = kv8::codes8<FMT>(v[i], iv); }
  if (tid == 0) { *k_scale = kv8::power_of_two(ek); *v_scale = kv8::power_of_two(ev); }
}

template <int D, int FMT, int HT>
__global__ void __launch_bounds__(Shape<D, HT>::NT, 2) attention_decode_kv8_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_v, Params p) {
  using S = Shape<D, HT>;
  constexpr int WARPS = S::WARPS, NT = S::NT, SLOTS = S::SLOTS, POS = S::POS;
  constexpr int NC = D / 16, MT = POS / 16;                 // 16-byte chunks of a row (steps of k, tiles of M); tiles of 16 positions
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint64_t full_bar[WARPS * SLOTS];
  __shared__ float wm[WARPS][HT * 8], wl[WARPS][HT * 8];
  __shared__ uint32_t top_s[16];
  __shared__ float2 ml_s[HT * 8];                           // this split's reference and sum per head, for the cluster
  __shared__ int abort_s;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  float* sums = reinterpret_cast<float*>(ring + S::MERGE);  // [G][D]: this split's outputs, for the cluster
  static_assert(S::RING >= S::MERGE + HT * 8 * D * 4, "room for the sums behind what the warps leave");
  const int split = blockIdx.x, kvh = blockIdx.y, t = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, j = lane & 3;
  volatile int* aborted = &abort_s;
  if (tid == 0) {
    for (int s = 0; s < WARPS * SLOTS; ++s) mbar_init(&full_bar[s], 1);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();                                          // the barriers are ready
  pdl_wait();
  pdl_launch_dependents();                                  // (in this order: it reads cached rows, see common.cuh)
  const int G = p.n_heads / p.n_kv_heads;
  const __nv_bfloat16* q = p.q + ((size_t)t * p.n_heads + (size_t)kvh * G) * D;
  uint2 raw[HT][NC];                                        // asked for before the indices, which are a chain of four reads
#pragma unroll
  for (int h = 0; h < HT; ++h)
#pragma unroll
    for (int c = 0; c < NC; ++c)
      raw[h][c] = h * 8 + g < G ? *reinterpret_cast<const uint2*>(q + (size_t)(h * 8 + g) * D + c * 16 + 4 * j) : make_uint2(0u, 0u);
  int pos = p.token_pos[t];
  const int seq = p.token_seq[t];
  int slot = seq >= 0 && seq < p.n_seqs ? p.seq_slot[seq] : -1;
  // a position below zero is a padded row: it sees nothing and its output is zero
  if (pos >= 0 && (slot < 0 || slot >= p.n_slots || pos / PAGE >= p.max_blocks)) {
    if (tid == 0 && p.error_flag) atomicExch(p.error_flag, kIndexOutside);
    pos = -1;
  }
  const int lo = pos < 0 ? 0 : window_low(p.window_kind, p.window_size, pos);
  const int* table = p.page_table + (size_t)max(slot, 0) * p.max_blocks;
  // The complete blocks that hold visible positions: kept ones (0 .. n_kept - 1), then the window's, b_lo .. own - 1.
  const int b_lo = lo / PAGE, own = pos < 0 ? 0 : pos / PAGE;
  const int keep = p.window_kind == 2 ? p.keep_first : 0;
  const int n_kept = min((keep + PAGE - 1) / PAGE, b_lo);
  const int n_items = pos < 0 ? 0 : n_kept + own - b_lo;
  auto block_of = [&](int i) { return i < n_kept ? i : b_lo + i - n_kept; };
  const int per = (n_items + kTailUnits + p.n_splits - 1) / p.n_splits;
  const int begin = min(n_items, split * per), end = split == p.n_splits - 1 ? n_items : min(n_items, begin + per);
  const bool has_tail = pos >= 0 && split == p.n_splits - 1;
  const int total_pages = p.n_pages;
  const size_t tail = ((size_t)max(slot, 0) * p.n_kv_heads + kvh) * (PAGE * D);

  // This warp's half pages are number warp, warp + WARPS, ... of the split's; its tiles y = 2 x (keys of its half page x), 2 x + 1 (values)
  const int halves = 2 * (end - begin);
  const int mine = max(0, (halves - warp + WARPS - 1) / WARPS);
  auto half_of = [&](int x) { return warp + x * WARPS; };
  auto block_at = [&](int x) { return block_of(begin + (half_of(x) >> 1)); };
  uint8_t* slots = ring + warp * SLOTS * S::TILE;
  uint64_t* bars = full_bar + warp * SLOTS;
  int ids = 0;                                              // page numbers of 32 of its half pages, one per lane, for the tiles asked for
  auto take_ids = [&](int x) {
    ids = x + lane < mine ? table[block_at(x + lane)] : 0;
    if (ids < 0 || ids >= total_pages) {                    // (beyond the map's last row: zeros arrive)
      ids = total_pages;
      if (p.error_flag) atomicExch(p.error_flag, kIndexOutside);
    }
  };
  auto ask = [&](int y, int at) {                           // tile y into slot `at` (all lanes call it)
    const int x = y >> 1;
    if (x >= mine) return;
    if (y % 64 == 0 && y > 0) take_ids(x);
    const int page = __shfl_sync(0xffffffffu, ids, x & 31);
    if (lane == 0) {
      mbar_expect_tx(&bars[at], S::TILE);
      tma_load_2d(slots + at * S::TILE, y & 1 ? &map_v : &map_k, &bars[at], 0,
                  ((page * p.n_kv_heads + kvh) * (PAGE / POS) + (half_of(x) & 1)) * S::LINES);
    }
  };
  take_ids(0);
#pragma unroll
  for (int y = 0; y < SLOTS; ++y) ask(y, y);

  {
    // the own block: four warps of the last split take 16 of its positions each
    const int tail0 = own * PAGE + warp * 16;
    const bool tail_any = has_tail && warp < 4 && tail0 <= pos && (tail0 + 15 >= lo || tail0 < keep);
    const __nv_bfloat16 *kt_tail = p.k_tail + tail + (warp & 3) * 16 * D, *vt_tail = p.v_tail + tail + (warp & 3) * 16 * D;
    uint4 tk[NC];                                           // rows g and g + 8, 16 bytes of each two chunks
    if (tail_any) {
#pragma unroll
      for (int c = 0; c < NC; c += 2) {
        tk[c] = *reinterpret_cast<const uint4*>(kt_tail + g * D + c * 16 + 8 * j);
        tk[c + 1] = *reinterpret_cast<const uint4*>(kt_tail + (g + 8) * D + c * 16 + 8 * j);
      }
    }
    // B operands: column g = head g of the tile (heads beyond the group are zeros), k in the order of a lane's bytes
    uint32_t qf[HT][NC][2];
    float f[HT][2];                                         // per head of this lane's columns 2j, 2j + 1: 2^(q's power)
#pragma unroll
    for (int h = 0; h < HT; ++h) {
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < NC; ++c) top = max(top, kv8::top_of(make_uint4(raw[h][c].x, raw[h][c].y, 0u, 0u)));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the largest element lies in [2^14, 2^15) after the division (below 2^-106: as it is, times 2^120)
      const int e = max(-120, (int)(top >> 7) - 127 - 14);
      const float inv = kv8::power_of_two(-e);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        qf[h][c][0] = pack_f16(kv8::lo_f32(raw[h][c].x) * inv, kv8::hi_f32(raw[h][c].x) * inv);
        qf[h][c][1] = pack_f16(kv8::lo_f32(raw[h][c].y) * inv, kv8::hi_f32(raw[h][c].y) * inv);
      }
      const float mine = kv8::power_of_two(e);
      f[h][0] = __shfl_sync(0xffffffffu, mine, 8 * j);
      f[h][1] = __shfl_sync(0xffffffffu, mine, 8 * j + 4);
    }
    float m[HT][2], l[HT][2], o[HT][NC][4];
#pragma unroll
    for (int h = 0; h < HT; ++h) {
      m[h][0] = m[h][1] = -1e30f;
      l[h][0] = l[h][1] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[h][c][0] = o[h][c][1] = o[h][c][2] = o[h][c][3] = 0.f;
    }
    // The maxima mx of new scores (base 2, the value scale's power in them) over this lane's positions: over all lanes of the
    // head, and the reference raised where they have outgrown it.
    auto raise = [&](float (&mx)[HT][2]) {
      bool grow = false;
#pragma unroll
      for (int h = 0; h < HT; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = mx[h][e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          mx[h][e] = x;
          grow |= x > m[h][e] + kSlack;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float now = fmaxf(m[h][e], mx[h][e]), by = ex2(m[h][e] - now);
            m[h][e] = now;
            l[h][e] *= by;
#pragma unroll
            for (int c = 0; c < NC; ++c) { o[h][c][e] *= by; o[h][c][e + 2] *= by; }
          }
      }
    };
    auto sees = [&](int kp) { return (kp >= lo || kp < keep) && kp <= pos; };
    // score -> base 2 with the value scale's power; `unit`: what a unit of s is worth, times the softmax scale
    auto scaled = [&](float s, float unit, float cap_unit, float ev) {
      return p.cap_out > 0.f ? fmaf(tanhf(s * cap_unit), p.cap_out, ev) : fmaf(s, unit, ev);
    };

    if (tail_any) {
      // the own block, in bfloat16 (its queries too)
      uint32_t tv[NC][4];                                   // value words of positions 2j, 2j + 1, 2j + 8, 2j + 9: zeros where masked
      bool in[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) in[r] = sees(tail0 + 2 * j + (r & 1) + (r >> 1) * 8);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          tv[c][r] = in[r] ? *reinterpret_cast<const uint32_t*>(vt_tail + (2 * j + (r & 1) + (r >> 1) * 8) * D + c * 16 + 2 * g) : 0u;
      float s[HT][4] = {}, mx[HT][2];
#pragma unroll
      for (int c = 0; c < NC; c += 2) {
        // a lane's 16 bytes of a row fill its places in two steps of k
        const uint4 x = tk[c], y = tk[c + 1];
        const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
        for (int h = 0; h < HT; ++h) {
          const uint4 b = h * 8 + g < G ? *reinterpret_cast<const uint4*>(q + (size_t)(h * 8 + g) * D + c * 16 + 8 * j)
                                        : make_uint4(0u, 0u, 0u, 0u);
          mma_bf16(s[h], a0, b.x, b.y);
          mma_bf16(s[h], a1, b.z, b.w);
        }
      }
      const bool in0 = sees(tail0 + g), in1 = sees(tail0 + g + 8);
#pragma unroll
      for (int h = 0; h < HT; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[h][e] = in0 ? scaled(s[h][e], p.scale_log2, p.cap_in, 0.f) : -INFINITY;
          s[h][e + 2] = in1 ? scaled(s[h][e + 2], p.scale_log2, p.cap_in, 0.f) : -INFINITY;
          mx[h][e] = fmaxf(s[h][e], s[h][e + 2]);
        }
      raise(mx);
      uint32_t b[HT][2];
#pragma unroll
      for (int h = 0; h < HT; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[h][e] = ex2(s[h][e] - (m[h][e & 1] - kLift));
          l[h][e & 1] += s[h][e];
        }
        b[h][0] = transposed(pack_bf16(s[h][0], s[h][1]));
        b[h][1] = transposed(pack_bf16(s[h][2], s[h][3]));
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint32_t a[4] = {__byte_perm(tv[c][0], tv[c][1], 0x5410), __byte_perm(tv[c][0], tv[c][1], 0x7632),
                               __byte_perm(tv[c][2], tv[c][3], 0x5410), __byte_perm(tv[c][2], tv[c][3], 0x7632)};
#pragma unroll
        for (int h = 0; h < HT; ++h) mma_bf16(o[h][c], a, b[h][0], b[h][1]);
      }
    }

    float ks_all = 0.f, ev_all = 0.f;
    int at = 0;                                             // the slot of the next tile
    uint32_t parity = 0;
    auto next = [&] { if (++at == SLOTS) { at = 0; parity ^= 1u; } };
    for (int x = 0; x < mine; ++x) {
      if (x % 32 == 0) {                                    // scales of the next 32 of its half pages, one per lane
        const int page = x + lane < mine ? table[block_at(x + lane)] : -1;
        const bool ok = page >= 0 && page < total_pages;
        ks_all = ok ? p.k_scale[(size_t)page * p.n_kv_heads + kvh] : 0.f;
        ev_all = ok ? log2f(fmaxf(p.v_scale[(size_t)page * p.n_kv_heads + kvh], 1e-30f)) : 0.f;      // (any scale is good)
      }
      const float ks = __shfl_sync(0xffffffffu, ks_all, x & 31), ev = __shfl_sync(0xffffffffu, ev_all, x & 31);
      const int first = block_at(x) * PAGE + (half_of(x) & 1) * POS;
      const bool ragged = first < lo && first + POS - 1 >= keep;            // (every position of a complete block is before pos)
      if (!__all_sync(0xffffffffu, mbar_wait(&bars[at], parity, aborted))) break;
      const uint32_t kt = smem_u32(slots + at * S::TILE);
      float s[HT][MT][4] = {};
      uint32_t w[2][MT][4];                                 // two chunks of every tile of positions; the next two are loaded meanwhile
      auto load_k = [&](int c) {                            // positions 0-7 and 8-15 of a tile, chunk c, then chunk c + 1
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) ldmatrix_x4(w[c >> 1 & 1][mt], kt + chunk_at<D>(mt * 16 + (lane & 15), c + (lane >> 4)));
      };
      load_k(0);
#pragma unroll
      for (int c = 0; c < NC; c += 2) {
        if (c + 2 < NC) load_k(c + 2);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t a[4];
            numbers<FMT, false>(w[c >> 1 & 1][mt][2 * u], a[0], a[2]);
            numbers<FMT, false>(w[c >> 1 & 1][mt][2 * u + 1], a[1], a[3]);
#pragma unroll
            for (int h = 0; h < HT; ++h) mma_f16(s[h][mt], a, qf[h][c + u][0], qf[h][c + u][1]);
          }
      }
      __syncwarp();                                         // every lane has its keys (they are in products): the slot is free
      ask(2 * x + SLOTS, at);
      next();
      const float v_inv = ex2(-ev);                         // (exact for a power of two)
      float mx[HT][2];
#pragma unroll
      for (int h = 0; h < HT; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float unit = f[h][e] * ks * p.scale_log2, cap_unit = f[h][e] * ks * p.cap_in;
          float top = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float y = scaled(s[h][mt][e + 2 * r], unit, cap_unit, ev);
              if (ragged && !sees(first + mt * 16 + g + 8 * r)) y = -INFINITY;
              s[h][mt][e + 2 * r] = y;
              top = fmaxf(top, y);
            }
          mx[h][e] = top;
        }
      raise(mx);
      uint32_t b[HT][MT][2];
#pragma unroll
      for (int h = 0; h < HT; ++h) {
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[h][mt][e] = ex2(s[h][mt][e] - (m[h][e & 1] - kLift));
            sum[e & 1] += s[h][mt][e];
          }
          b[h][mt][0] = transposed(pack_f16(s[h][mt][0], s[h][mt][1]));
          b[h][mt][1] = transposed(pack_f16(s[h][mt][2], s[h][mt][3]));
        }
        l[h][0] = fmaf(sum[0], v_inv, l[h][0]);
        l[h][1] = fmaf(sum[1], v_inv, l[h][1]);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&bars[at], parity, aborted))) break;
      const uint32_t vt = smem_u32(slots + at * S::TILE);
      if (ragged) {
        // value rows that the query does not see become zeros (e4m3 may hold a NaN there): a row a lane
#pragma unroll 1
        for (int c = 0; c < NC; ++c)
          if (!sees(first + lane)) *reinterpret_cast<uint4*>(slots + at * S::TILE + chunk_at<D>(lane, c)) = make_uint4(0u, 0u, 0u, 0u);
        __syncwarp();
      }
      auto load_v = [&](int c) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) ldmatrix_x4_trans(w[c >> 1 & 1][mt], vt + chunk_at<D>(mt * 16 + (lane & 15), c + (lane >> 4)));
      };
      load_v(0);
#pragma unroll
      for (int c = 0; c < NC; c += 2) {
        if (c + 2 < NC) load_v(c + 2);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t a[4];
            numbers<FMT, true>(w[c >> 1 & 1][mt][2 * u], a[0], a[1]);
            numbers<FMT, true>(w[c >> 1 & 1][mt][2 * u + 1], a[2], a[3]);
#pragma unroll
            for (int h = 0; h < HT; ++h) mma_f16(o[h][c + u], a, b[h][mt][0], b[h][mt][1]);
          }
      }
      // the zeros written above must be ordered before the copy engine writes this slot again
      if (ragged) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      ask(2 * x + 1 + SLOTS, at);
      next();
    }
    // l is a sum over this lane's positions: complete it over the lanes with the same heads
#pragma unroll
    for (int h = 0; h < HT; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], 4);
        l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], 8);
        l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], 16);
      }
    // every warp is done with its slots; all of them go on, or none
    if (!__syncthreads_or(*aborted)) {
      float* mo = reinterpret_cast<float*>(ring);           // [warps][heads][D]
#pragma unroll
      for (int h = 0; h < HT; ++h) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<float2*>(mo + ((size_t)(warp * HT + h) * 8 + 2 * j + e) * D + c * 16 + 2 * g) = make_float2(o[h][c][e], o[h][c][e + 2]);
        if (g == 0)
#pragma unroll
          for (int e = 0; e < 2; ++e) { wm[warp][h * 8 + 2 * j + e] = m[h][e]; wl[warp][h * 8 + 2 * j + e] = l[h][e]; }
      }
      __syncthreads();
      if (tid < G) {                                        // a thread per head: the warps' weights (in wm), the sum (in wl[0])
        const int head = kvh * G + tid;
        float M = -1e30f, L = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, wm[w][tid]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float by = exp2f(wm[w][tid] - M);
          L += by * wl[w][tid];
          wm[w][tid] = by;
        }
        if (p.n_splits == 1) {
          L += sink_term(p.sink, head, M);
          wl[0][tid] = L == 0.f ? 0.f : 1.f / L;
        } else if (p.clustered) {
          ml_s[tid] = make_float2(M, L);
        } else {
          p.part_ml[((size_t)t * p.n_heads + head) * p.n_splits + split] = make_float2(M, L);
        }
      }
      __syncthreads();
      for (int idx = tid; idx < G * D / 2; idx += NT) {
        const int h = idx / (D / 2), d = idx % (D / 2) * 2, head = kvh * G + h;
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float2 x = *reinterpret_cast<const float2*>(mo + (size_t)(w * HT * 8 + h) * D + d);
          const float by = wm[w][h];
          acc.x = fmaf(by, x.x, acc.x);
          acc.y = fmaf(by, x.y, acc.y);
        }
        if (p.n_splits == 1) {
          const float inv = wl[0][h];
          *reinterpret_cast<uint32_t*>(p.out + ((size_t)t * p.n_heads + head) * D + d) = pack_bf16(acc.x * inv, acc.y * inv);
        } else if (p.clustered) {
          *reinterpret_cast<float2*>(sums + h * D + d) = acc;
        } else {
          *reinterpret_cast<float2*>(p.part_o + (((size_t)t * p.n_heads + head) * p.n_splits + split) * D + d) = acc;
        }
      }
    }
  }
  if (p.clustered) {
    // The splits' sums, each in its block's shared memory: every block joins a share of the outputs.  (All threads of all blocks
    // pass both barriers, whatever has happened before.)
    cluster_sync();
    const int rank = (int)cluster_rank(), n = p.n_splits;
    for (int i = rank + n * tid; i < G * D / 2; i += n * NT) {
      const int h = i / (D / 2), d = i % (D / 2) * 2, head = kvh * G + h;
      const uint32_t at = smem_u32(sums + h * D + d), ml_at = smem_u32(&ml_s[h]);
      float2 ml[kMaxCluster], v[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        ml[r] = r < n ? peer_pair(ml_at, r) : make_float2(-1e30f, 0.f);
        v[r] = r < n ? peer_pair(at, r) : make_float2(0.f, 0.f);
      }
      float M = -1e30f, L = 0.f;
      float2 acc = make_float2(0.f, 0.f);
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) M = fmaxf(M, ml[r].x);
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        const float by = exp2f(ml[r].x - M);
        L += by * ml[r].y;
        acc.x = fmaf(by, v[r].x, acc.x);
        acc.y = fmaf(by, v[r].y, acc.y);
      }
      L += sink_term(p.sink, head, M);
      const float inv = L == 0.f ? 0.f : 1.f / L;
      *reinterpret_cast<uint32_t*>(p.out + ((size_t)t * p.n_heads + head) * D + d) = pack_bf16(acc.x * inv, acc.y * inv);
    }
    cluster_sync();                                         // nobody leaves while its shared memory is read
  }
  if (has_tail && pos % PAGE == PAGE - 1) {
    // the block is complete: its codes and scales, for later steps (nobody reads that page in this one)
    const int page = table[own];
    if (page >= 0 && page < total_pages) {
      const size_t to = (size_t)page * p.n_kv_heads + kvh;
      hold_tail<D, FMT, NT>(p.k_tail + tail, p.v_tail + tail, p.k + to * (PAGE * D), p.v + to * (PAGE * D), p.k_scale_w + to, p.v_scale_w + to, top_s);
    } else if (tid == 0 && p.error_flag) {
      atomicExch(p.error_flag, kIndexOutside);
    }
  }
  if (*aborted) {
    // a wait ran out: say so, give the copies in flight time to land before the shared memory is released
    if (lane == 0 && p.error_flag) atomicExch(p.error_flag, 1);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
}

// out[t, h] = sum_s w_s O_s / sum_s w_s L_s, w_s = 2^(m_s - max m): a block per (token, head), a thread per feature.
template <int D>
__global__ void __launch_bounds__(D) attention_decode_kv8_combine(const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                                                                  __nv_bfloat16* __restrict__ out, int n_splits, const float* __restrict__ sink,
                                                                  int n_heads) {
  __shared__ float w_s[kMaxSplits];
  __shared__ float red[D / 32];
  const int tid = threadIdx.x;
  const size_t th = blockIdx.x;
  const float2* ml = part_ml + th * n_splits;
  const float* po = part_o + th * n_splits * D;
  pdl_wait();
  pdl_launch_dependents();
  float M = -1e30f, L = 0.f, acc = 0.f;
  if (n_splits <= 16) {
    // every thread takes all pairs and its own feature of every part at once: one trip to the L2, no barrier
    float2 a[16];
    float v[16];
#pragma unroll
    for (int s = 0; s < 16; ++s) {
      a[s] = s < n_splits ? __ldcg(ml + s) : make_float2(-1e30f, 0.f);
      v[s] = s < n_splits ? __ldcg(po + (size_t)s * D + tid) : 0.f;
    }
#pragma unroll
    for (int s = 0; s < 16; ++s) M = fmaxf(M, a[s].x);
#pragma unroll
    for (int s = 0; s < 16; ++s) {
      const float by = exp2f(a[s].x - M);
      L += by * a[s].y;
      acc += by * v[s];
    }
  } else {
    for (int s = tid; s < n_splits; s += D) M = fmaxf(M, __ldcg(ml + s).x);
    M = warp_max(M);
    if ((tid & 31) == 0) red[tid >> 5] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < D / 32; ++w) M = fmaxf(M, red[w]);
    __syncthreads();
    for (int s = tid; s < n_splits; s += D) {
      const float2 a = __ldcg(ml + s);
      const float by = exp2f(a.x - M);
      w_s[s] = by;
      L += by * a.y;
    }
    L = block_sum(L, red);                                  // (its barriers also publish w_s)
    for (int s0 = 0; s0 < n_splits; s0 += 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = s0 + i < n_splits ? __ldcg(po + (size_t)(s0 + i) * D + tid) : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s0 + i < n_splits) acc += w_s[s0 + i] * v[i];
    }
  }
  L += sink_term(sink, (int)(th % n_heads), M);
  out[th * D + tid] = __float2bfloat16_rn(L == 0.f ? 0.f : acc / L);
}

template <int D, int FMT, int HT>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int n_tokens, cudaStream_t stream) {
  auto* kernel = attention_decode_kv8_kernel<D, FMT, HT>;
  using S = Shape<D, HT>;
  constexpr int SMEM = S::SMEM;
  static bool ready[64] = {};                               // per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess) {
      cudaGetLastError();
      set_error("attention_decode_kv8: cannot reserve %d bytes of shared memory", SMEM);
      return 1;
    }
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n_splits, p.n_kv_heads, n_tokens);
  cfg.blockDim = dim3(S::NT);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.n_splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.clustered ? 2 : 1;
  count_launch();
  cudaLaunchKernelEx(&cfg, kernel, mk, mv, p);
  if (check_launch("attention_decode_kv8")) return 2;
  if (p.n_splits > 1 && !p.clustered) {
    cpi::launch_pdl(attention_decode_kv8_combine<D>, n_tokens * p.n_heads, D, 0, stream, p.part_o, p.part_ml, p.out, p.n_splits, p.sink,
                    p.n_heads);
    return check_launch("attention_decode_kv8_combine");
  }
  return 0;
}

}  // namespace dec8
}  // namespace cpi

using namespace cpi;

extern "C" int cpi_attention_decode_kv8_supported(int n_heads, int n_kv_heads, int head_dim, int page_size) {
  if (n_kv_heads <= 0 || n_heads % n_kv_heads) return 0;
  return (head_dim == 64 || head_dim == 128) && page_size == kv8::PAGE && n_heads / n_kv_heads <= 16 && n_kv_heads <= 65535;
}

// Whether `n_splits` blocks of threads for each of `base` (token, kv head) pairs are joined within the kernel, as clusters, or
// through scratch by a second one.  A cluster saves a launch and the scratch, but its blocks stay until the last of them is
// through: 160 blocks (5 windowed sequences, 8 kv heads of 64) take 7.9 us as clusters and 8.1 with the second kernel, 256 (8 x 4,096
// positions, 8 kv heads of 128) 23.8 and 22.5, 1,536 (64 sequences) 203 and 190.
extern "C" int cpi_attention_decode_kv8_clustered(int base, int n_splits) {
  return n_splits > 1 && n_splits <= dec8::kMaxCluster && 3l * base * n_splits <= 4l * sm_count();
}

// Blocks of threads that share an SM, for the caller's choice of `n_splits`.
extern "C" int cpi_attention_decode_kv8_blocks_per_sm() { return 2; }

// q, out [T, NH, D] bfloat16, one token per sequence; codes k, v [n_pages, NKV, 64, D]; `fmt` 0 int8, 1 e4m3.  `scratch`:
// T * NH * splits * (D + 2) floats, 8-byte aligned (none if they are joined in the kernel).
extern "C" int cpi_attention_decode_kv8(const void* q, void* out, void* k, void* v, float* k_scale, float* v_scale, int n_pages,
                                        const void* k_tail, const void* v_tail, int n_slots, const int* page_table, int max_blocks,
                                        const int* token_seq, const int* token_pos, const int* seq_slot, int n_seqs, int n_tokens, int n_heads,
                                        int n_kv_heads, int head_dim, int fmt, int window_kind, int window_size, int keep_first, float scale,
                                        float softcap, const float* sink, int n_splits, float* scratch, int* error_flag, cudaStream_t stream) {
  if (n_tokens == 0) return 0;
  CPI_REQUIRE(cpi_attention_decode_kv8_supported(n_heads, n_kv_heads, head_dim, kv8::PAGE),
              "attention_decode_kv8: unsupported shape (heads %d/%d, head size %d)", n_heads, n_kv_heads, head_dim);
  CPI_REQUIRE(fmt == kv8::kInt8 || fmt == kv8::kE4m3, "attention_decode_kv8: unknown format %d", fmt);
  CPI_REQUIRE(window_kind == 0 || window_size > 0, "attention_decode_kv8: window kind %d needs a size > 0", window_kind);
  CPI_REQUIRE(n_splits >= 1 && n_splits <= dec8::kMaxSplits && n_tokens <= 65535, "attention_decode_kv8: bad grid (%d splits of at most %d, %d tokens)",
              n_splits, dec8::kMaxSplits, n_tokens);
  // Without scratch the splits are joined in the kernel (see cpi_attention_decode_kv8_clustered).
  const bool clustered = n_splits > 1 && !scratch;
  CPI_REQUIRE(!clustered || n_splits <= dec8::kMaxCluster, "attention_decode_kv8: split scratch is missing");
  // the codes as lines of 128 bytes: a tile of 32 positions of a head is 32 * D / 128 of them
  CUtensorMap mk, mv;
  const uint64_t lines = (uint64_t)n_pages * n_kv_heads * (kv8::PAGE * head_dim / 128);
  CPI_REQUIRE(n_pages > 0 && lines + (uint64_t)n_kv_heads * kv8::PAGE < (1ull << 31), "attention_decode_kv8: a cache of %d pages of %d heads", n_pages, n_kv_heads);
  if (tc::get_map_2d_bf16(k, 64, lines, 128, 64, 32 * head_dim / 128, &mk)) return 1;
  if (tc::get_map_2d_bf16(v, 64, lines, 128, 64, 32 * head_dim / 128, &mv)) return 1;
  const long parts = (long)n_tokens * n_heads * n_splits;
  dec8::Params p{(const __nv_bfloat16*)q, (__nv_bfloat16*)out, k_scale, v_scale, (const __nv_bfloat16*)k_tail, (const __nv_bfloat16*)v_tail,
                 (uint8_t*)k, (uint8_t*)v, k_scale, v_scale, page_table, max_blocks, n_pages, n_slots, n_seqs, token_seq, token_pos, seq_slot,
                 n_heads, n_kv_heads, window_kind, window_size, keep_first > 0 ? keep_first : 0, scale * 1.4426950408889634f,
                 softcap > 0.f ? scale / softcap : 0.f, softcap > 0.f ? softcap * 1.4426950408889634f : 0.f, n_splits, clustered,
                 scratch, scratch ? reinterpret_cast<float2*>(scratch + parts * head_dim) : nullptr, sink, error_flag};
  const bool wide = n_heads / n_kv_heads > 8;
#define CPI_DEC8(D, F) (wide ? dec8::launch<D, F, 2>(mk, mv, p, n_tokens, stream) : dec8::launch<D, F, 1>(mk, mv, p, n_tokens, stream))
  if (head_dim == 128) return fmt ? CPI_DEC8(128, 1) : CPI_DEC8(128, 0);
  return fmt ? CPI_DEC8(64, 1) : CPI_DEC8(64, 0);
#undef CPI_DEC8
}
CPI_PACKED(cpi_attention_decode_kv8)
