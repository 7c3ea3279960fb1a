// The cache in 8 bits (kv8.cuh) around a step of several tokens: the pages that its attention reads.
//
// The attention of a prompt reads bfloat16 pages of the step's own: `earlier` pages hold the numbers that complete blocks stand
// for, `exact` pages the blocks that the step's tokens fall into, as projected (the projection has stored the new rows there).
// One launch does what is left, a job per page, a block of threads per (page, head, keys or values):
//   earlier block   its codes and scale -> the numbers they stand for
//   own block       rows before the step's first come from the sequence's tail, rows behind its last become zero; if the block is
//                   complete, its codes and scale go to the cache and the numbers they stand for to its `earlier` page
//   tail            the sequence's last block, if it is not complete, is copied to the tail by the threads that have read the
//                   tail before (the sequence's first own block), so no other block of threads can still want the old rows
// Bound by bytes: an earlier block reads 1 byte and writes 2 per element, an own block reads 2 and writes 3.
#include "kv8.cuh"
#include "packed.cuh"

namespace cpi {
namespace kv8 {

constexpr int kJobWords = 8;
struct StageParams {
  const int* jobs;                         // [n_jobs, 8]: slot, block, first new row, rows, earlier page, exact page, last page, last rows
  const int* page_table; int max_blocks;   // pages of the cache, per slot and block
  int n_pages, n_slots, n_step_pages, n_kv_heads;
  uint8_t *k, *v; float *k_scale, *v_scale;         // [n_pages, kv heads, 64, D], [n_pages, kv heads]
  __nv_bfloat16 *k_tail, *v_tail;                   // [n_slots, kv heads, 64, D]
  __nv_bfloat16 *k_pages, *v_pages;                 // [n_step_pages, kv heads, 64, D]
  int* error_flag;
};

template <int D, int FMT>
__global__ void __launch_bounds__(256) kv8_stage_kernel(StageParams p) {
  constexpr int VEC = PAGE * D / 8, PER = VEC / 256;        // vectors of eight numbers in a (page, head) tile, per thread
  __shared__ uint32_t red[8];
  const int tid = threadIdx.x, head = blockIdx.y, values = blockIdx.z;
  pdl_wait();
  pdl_launch_dependents();
  __nv_bfloat16* step_pages = values ? p.v_pages : p.k_pages;
  float* scales = values ? p.v_scale : p.k_scale;
  const int* job = p.jobs + (size_t)blockIdx.x * kJobWords;
  const int slot = job[0], block = job[1], r0 = job[2], r1 = job[3], earlier = job[4], exact = job[5], last = job[6], last_rows = job[7];
  if (slot < 0 || slot >= p.n_slots || block < 0 || block >= p.max_blocks) {
    if (tid == 0 && p.error_flag) atomicExch(p.error_flag, kIndexOutside);
    return;
  }
  const int page = p.page_table[(size_t)slot * p.max_blocks + block];
  if (page < 0 || page >= p.n_pages) {
    if (tid == 0 && p.error_flag) atomicExch(p.error_flag, kIndexOutside);
    return;
  }
  const size_t cache_tile = ((size_t)page * p.n_kv_heads + head) * (PAGE * D), scale_at = (size_t)page * p.n_kv_heads + head;
  auto step_tile = [&](int pg) { return step_pages + ((size_t)pg * p.n_kv_heads + head) * (PAGE * D); };
  uint8_t* codes = (values ? p.v : p.k) + cache_tile;
  if (exact < 0) {                                          // an earlier block
    const float s = scales[scale_at];
    uint4* dst = reinterpret_cast<uint4*>(step_tile(earlier));
    uint2 c[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) c[i] = reinterpret_cast<const uint2*>(codes)[tid + i * 256];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint2 a = values4<FMT>(c[i].x, s), b = values4<FMT>(c[i].y, s);
      dst[tid + i * 256] = make_uint4(a.x, a.y, b.x, b.y);
    }
    return;
  }
  __nv_bfloat16* tail = (values ? p.v_tail : p.k_tail) + ((size_t)slot * p.n_kv_heads + head) * (PAGE * D);
  uint4* own = reinterpret_cast<uint4*>(step_tile(exact));
  uint4 v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = tid + i * 256, row = at / (D / 8);
    if (row >= r1) own[at] = v[i] = make_uint4(0, 0, 0, 0);
    else if (row < r0) own[at] = v[i] = reinterpret_cast<const uint4*>(tail)[at];
    else v[i] = own[at];
  }
  if (last >= 0 && last_rows < PAGE) {                      // this job keeps the tail: the sequence's newest block
    const uint4* src = reinterpret_cast<const uint4*>(step_tile(last));
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = tid + i * 256, row = at / (D / 8);
      if (row < last_rows && (last != exact || row >= r0)) reinterpret_cast<uint4*>(tail)[at] = last == exact ? v[i] : src[at];
    }
  }
  if (r1 < PAGE) return;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) top = max(top, top_of(v[i]));
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = max(top, red[w]);
  const int e = scale_exponent<FMT>(__uint_as_float(top << 16));
  const float s = power_of_two(e), inv = power_of_two(-e);
  if (tid == 0) scales[scale_at] = s;
  uint4* dst = reinterpret_cast<uint4*>(step_tile(max(earlier, 0)));
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint2 c = codes8<FMT>(v[i], inv);
    reinterpret_cast<uint2*>(codes)[tid + i * 256] = c;
    if (earlier >= 0) {
      const uint2 a = values4<FMT>(c.x, s), b = values4<FMT>(c.y, s);
      dst[tid + i * 256] = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
}

}  // namespace kv8
}  // namespace cpi

using namespace cpi;

// `fmt`: 0 int8, 1 e4m3.  Pointers are 16-byte aligned; head_dim 64 or 128; pages of 64 positions.
extern "C" int cpi_kv8_stage(const int* jobs, int n_jobs, const int* page_table, int max_blocks, int n_slots, void* k, void* v, float* k_scale,
                             float* v_scale, int n_pages, void* k_tail, void* v_tail, void* k_pages, void* v_pages, int n_step_pages,
                             int n_kv_heads, int head_dim, int fmt, int* error_flag, cudaStream_t stream) {
  if (n_jobs == 0) return 0;
  CPI_REQUIRE(head_dim == 64 || head_dim == 128, "kv8_stage: head size %d (64 or 128)", head_dim);
  CPI_REQUIRE(fmt == kv8::kInt8 || fmt == kv8::kE4m3, "kv8_stage: unknown format %d", fmt);
  CPI_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 65535, "kv8_stage: %d key/value heads", n_kv_heads);
  kv8::StageParams p{jobs, page_table, max_blocks, n_pages, n_slots, n_step_pages, n_kv_heads, (uint8_t*)k, (uint8_t*)v, k_scale, v_scale,
                     (__nv_bfloat16*)k_tail, (__nv_bfloat16*)v_tail, (__nv_bfloat16*)k_pages, (__nv_bfloat16*)v_pages, error_flag};
  dim3 grid(n_jobs, n_kv_heads, 2);
  auto* kernel = head_dim == 128 ? (fmt ? kv8::kv8_stage_kernel<128, 1> : kv8::kv8_stage_kernel<128, 0>)
                                 : (fmt ? kv8::kv8_stage_kernel<64, 1> : kv8::kv8_stage_kernel<64, 0>);
  cpi::launch_pdl(kernel, grid, 256, 0, stream, p);
  return check_launch("kv8_stage");
}
CPI_PACKED(cpi_kv8_stage)
