// Prefill attention over the cache in 8 bits (kv8.cuh) on tcgen05: two tiles of 128 queries of one head against the pages of a step.
//
// A query sees its own block of 64 positions as projected and earlier blocks as the numbers they are held as; both stand in
// bfloat16 pages of the step's own, named by two tables (kv8_stage has made them).  A block of threads takes up to 256 consecutive
// tokens of one sequence and one query head, query tile A (the first 128 rows) and B (the rest), as in attention_prefill.cu: warp 8
// streams key/value tiles of 128 positions (two pages, TMA with the 128-byte swizzle) into a ring of five slots, K(i), V(i),
// K(i+1), ...; one lane of warp 9 issues the MMAs, alternating between A and B, so that the tensor pipe works for one while the
// other's softmax runs:
//     S = Q K^T            both operands K-major from shared memory, S in tensor memory
//     P = 2^(S*c - m)      as bfloat16 over columns of the S it came from
//     O += P V             P as the A operand from tensor memory, V consumed MN-major from the page layout [position][dim]
//
// The axis of key tiles begins with the exact tiles of A (those that hold its own blocks), goes on with the earlier blocks' and ends
// with the exact tiles of B: A meets a prefix of it and B a suffix.  A row's mask is that of the window cut at the start of its block,
// from one side or the other.  Pages that a tile does not have are asked for beyond the tensor's end and arrive as zeros, rows behind
// the newest position are zero already: nothing is overwritten in shared memory.  A masked weight is a zero in the product P V, so a
// value that is not finite also reaches queries of its sequence that do not see it, in the same key tile.  Per query tile that is one or
// two key tiles more than over a cache in bfloat16 (they hold the own blocks twice).
//
// Softmax: warps 0-3 own query tile A, warps 4-7 tile B; thread r of a group owns query row r and all 128 columns of a tile.  A row's
// reference m is its first tile's maximum, raised (and O rescaled in tensor memory) only when the row maximum has outgrown it by
// 2^40: P is bfloat16 and the sums are float32, which have the same range of powers, so nothing is lost by numbers up to 2^40 (sums up
// to 2^57, outputs finite for values up to 2^70), and it happens in a row's first tile and hardly ever again (keys and queries with a
// few large features, 3,001 tokens of 40 heads: 190 us with 2^8, 171 with 2^40).  P has 8 bits because the A operand of a product
// with bfloat16 values is bfloat16: outputs are off by 0.0021 to 0.0023 of their size where rounding the output alone takes 0.0016
// (the rest of P as a second operand would double the value products); row sums take the weights unrounded.
// Tiles without a mask are taken into registers whole, the maximum first, then P and the sum with two numbers to an instruction.
// Masked tiles, and those that outgrow a reference, go by 32 columns with the next ones on their way, against the reference they
// have; what has been stored of a tile's P is rescaled
// too.  Columns that no row of the warp sees are passed over.
//
// Bound by the chain S -> softmax -> P V -> next S of each query tile (about 3,600 cycles for two tiles of 128 x 128, where the products
// take 2,048 and the exponentials as many) and by a block's start and end, which nothing hides (6,000 cycles from its first
// instruction to its first S: indices, page numbers, loads; 3,000 at the end).  3,001 tokens of 40/8 heads of 128: 122 us (757 TFLOP/s).
// The way there: 149 with one number to an instruction, masked and first tiles in two passes, and each thread writing its own row 16
// bytes at a time (8,000 cycles a block); two numbers to an instruction and the maximum of three 146; rows written as whole lines
// 135; masked tiles in one pass and first tiles, if nothing is masked, from registers 123.  What was tried beside it: two threads
// to a row, sixteen warps, either spill with 96 registers each or read S twice; P
// handed on in two halves (the issuing warp then waits for one tile's second half while the other's is ready); every tile by 32
// columns (a vote each; 141); one S for both query tiles, read into registers at once, with the score products two steps ahead (145:
// the issuing warp's waits, 200 cycles each behind the exponentials of the warps beside it, leave the pipe idle); 224 registers for
// the softmax warps (126): all slower.  A quarter of the exponentials as cubics on the multipliers takes 2% off and is not taken: it is
// 7e-5 off and what is not finite would need a path of its own.
//
// Few query tiles over many keys share their key tiles out among blocks of threads (n_splits), joined by a second kernel.
// Every mbarrier wait is bounded; when one runs out the block sets *error_flag and leaves.
#include "prefill_tc.cuh"
#include "f32x2.cuh"
#include "packed.cuh"
#include <type_traits>

namespace cpi {
namespace pre8 {

using namespace pre;

constexpr int PAGE = 64;
constexpr int kRingSlots = 5;           // key and value tiles in shared memory at a time
constexpr int kSoftmaxWarps = 8, kThreads = (kSoftmaxWarps + 2) * 32;
constexpr float kWideSlack = 40.0f;

struct Params {
  __nv_bfloat16* out;                 // [T, NH * D]
  const int *earlier_table, *exact_table; int width;      // pages by sequence of the step and block, -1: none
  const int *token_pos, *token_seq;
  const int *tile_tok0, *tile_rows;   // per query tile: first packed token, valid rows
  int n_heads, n_kv_heads;
  int window_kind, window_size, keep_first;
  float scale_log2;
  int* error_flag;
  const float* sink;                  // [NH] float32 or null: exp(sink[h]) joins the softmax denominator (no key, no value)
  float cap_in, cap_out;              // soft cap c > 0 on the scaled scores: cap_in = scale / c, cap_out = c log2(e); else 0
  int n_pages, n_tokens, n_seqs;
  int n_splits;                       // blocks of threads that share a query tile's axis of key tiles
  float* part_o; float2* part_ml;     // with several: [T, NH, splits, D] sums, [T, NH, splits] reference and row sum
};

// As mbar_wait, with one look that does not suspend the thread first.
__device__ __forceinline__ bool wait_soon(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0 || mbar_wait(bar, parity, abort_flag);
}
// The largest of three (a NaN is passed over).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The loads issued so far have landed in these registers (named, so that nothing reads them before).
__device__ __forceinline__ void landed32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
        "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
        "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :: "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  tmem_ld16_issue(taddr, r);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
}
template <int D, bool CAPPED>
__global__ void __launch_bounds__(kThreads, 1) attention_prefill_kv8_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                         const __grid_constant__ CUtensorMap map_k,
                                                                         const __grid_constant__ CUtensorMap map_v, Params p) {
  constexpr int HALVES = D / 64;                       // 64-element (128-byte) column blocks of a row
  constexpr uint32_t HALF_BYTES = 128 * 128;           // 128 rows x 128 bytes
  constexpr uint32_t Q_BYTES = HALVES * HALF_BYTES;    // one query tile of 128 rows
  constexpr uint32_t KV_BYTES = HALVES * HALF_BYTES;   // one of K or V, 128 positions
  constexpr uint32_t TMEM_COLS = 512;                  // S of tile A, S of tile B (128 columns each), O of A, O of B
  constexpr int NSLOT = kRingSlots;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t q_full, kv_full[NSLOT], kv_empty[NSLOT], s_full[2], p_full[2], o_done[2];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* q_s = smem_raw;                             // [2 query tiles]
  uint8_t* ring = q_s + 2 * Q_BYTES;                   // [NSLOT]

  if (tid == 0) {
    mbar_init(&q_full, 1);
    for (int s = 0; s < NSLOT; ++s) { mbar_init(&kv_full[s], 1); mbar_init(&kv_empty[s], 1); }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4); mbar_init(&o_done[s], 1);
    }
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  pdl_wait();
  pdl_launch_dependents();                              // (in this order, and not before the tensor memory is ours: see common.cuh)
  const int tile = blockIdx.y, head = blockIdx.x;       // heads are the fast axis: all heads of the longest tile start first
  const int kvh = head / (p.n_heads / p.n_kv_heads);
  int tok0 = p.tile_tok0[tile], rows = p.tile_rows[tile];
  {                                                     // indices outside of the step: somewhere within it, and the error flag
    const bool good = tok0 >= 0 && tok0 < p.n_tokens && rows >= 1 && rows <= kTileRows && rows <= p.n_tokens - tok0;
    tok0 = min(max(tok0, 0), p.n_tokens - 1);
    rows = min(max(rows, 1), min(kTileRows, p.n_tokens - tok0));
    if (!good && tid == 0 && p.error_flag) atomicExch(p.error_flag, kIndexOutside);
  }
  if (warp == kSoftmaxWarps && lane == 0) {               // the queries of both tiles, under the reads of what else there is to know
    mbar_expect_tx(&q_full, Q_BYTES * (rows > BQ ? 2 : 1));
    for (int x = 0; x < (rows > BQ ? 2 : 1); ++x)
      for (int h = 0; h < HALVES; ++h)
        tma_load_2d(q_s + x * Q_BYTES + h * HALF_BYTES, &map_q, &q_full, head * D + h * 64, tok0 + x * BQ);
  }
  int seq = p.token_seq[tok0];
  // the tile's rows are consecutive positions of one sequence; rows 0-127 are query tile A, the rest tile B
  int pos_first = p.token_pos[tok0];
  if (seq < 0 || seq >= p.n_seqs || pos_first < 0 || pos_first > p.width * PAGE - rows) {
    seq = 0;
    pos_first = 0;
    if (tid == 0 && p.error_flag) atomicExch(p.error_flag, kIndexOutside);
  }
  const int pos_last = pos_first + rows - 1;
  const int rows_x[2] = {min(rows, BQ), max(rows - BQ, 0)};
  const bool has_b = rows_x[1] > 0;
  const int p0_x[2] = {pos_first, pos_first + BQ};                         // first position of A, of B
  const int p1_x[2] = {pos_first + rows_x[0] - 1, pos_last};               // last position of A, of B
  // key tiles (of 128 positions) that each query tile meets; the window's low end never decreases with the position
  const int kb_phys[2] = {window_low(p.window_kind, p.window_size, p0_x[0]) / BKV,
                          has_b ? window_low(p.window_kind, p.window_size, p0_x[1]) / BKV : 0};
  // Kept first positions: the key tiles that hold them and lie wholly below the window's first tile come first.
  // The loops below count key tiles on an axis of their own, `n_kept` kept tiles (key tiles 0 .. n_kept - 1) and
  // then the window's tiles without a gap: tile kt of the axis is key tile kt + (kt < n_kept ? 0 : gap).  With
  // kept positions both query tiles meet every tile of the axis from its start, which always holds position 0: the
  // second query tile sees kept positions also in the tiles between the two windows' first tiles (a tile of which
  // it sees nothing is masked whole: at most one).
  const int keep = p.window_kind == 2 ? p.keep_first : 0;
  const int n_kept = min((keep + BKV - 1) / BKV, kb_phys[0]);
  const int gap = kb_phys[0] - n_kept;
  // exact tiles of A, then earlier blocks' tiles up to the one that holds the last position before A's (B's) last
  // row's block, then exact tiles of B
  const int first_exact[2] = {p0_x[0] / BKV, p0_x[1] / BKV};
  const int n_exact[2] = {p1_x[0] / BKV - first_exact[0] + 1, has_b ? p1_x[1] / BKV - first_exact[1] + 1 : 0};
  auto tiles_to = [&](int x) { return max((p1_x[x] / PAGE * PAGE + BKV - 1) / BKV - gap, 0); };
  const int n_earlier = tiles_to(has_b ? 1 : 0);
  int kb_x[2] = {0, n_exact[0] + (has_b && keep == 0 ? kb_phys[1] - gap : 0)};
  int ke_x[2] = {n_exact[0] + tiles_to(0), has_b ? n_exact[0] + n_earlier + n_exact[1] : 0};
  int kt0 = 0, kt1 = has_b ? ke_x[1] : ke_x[0];                           // the union: every tile in it is met by A or B
  if (p.n_splits > 1) {                                        // this block's share of the union
    const int per = (kt1 + p.n_splits - 1) / p.n_splits;
    kt0 = min(kt1, (int)blockIdx.z * per);
    kt1 = min(kt1, kt0 + per);
#pragma unroll
    for (int x = 0; x < 2; ++x) { kb_x[x] = min(max(kb_x[x], kt0), kt1); ke_x[x] = max(min(ke_x[x], kt1), kb_x[x]); }
  }
  auto is_exact = [&](int kt) { return kt < n_exact[0] || kt >= n_exact[0] + n_earlier; };
  auto key_tile = [&](int kt) {
    if (kt < n_exact[0]) return first_exact[0] + kt;
    kt -= n_exact[0];
    if (kt >= n_earlier) return first_exact[1] + kt - n_earlier;
    return kt < n_kept ? kt : kt + gap;
  };
  const uint32_t tmem_s = tmem_base_s, tmem_o = tmem_base_s + 256;        // + 128 for tile B, both
  volatile int* abort_flag = &abort_s;
  bool ok = true;

  if (warp == kSoftmaxWarps) {
    if (lane == 0) {
      // ---- TMA producer: K(kt0), V(kt0), K(kt0 + 1), ... through the ring ----
      int n = 0;                                         // item of the ring: 2 (kt - kt0) for keys, + 1 for values
      for (int kt = kt0; kt < kt1 && ok; ++kt) {
        const int blk0 = key_tile(kt) * (BKV / PAGE);
        const int* pages = (is_exact(kt) ? p.exact_table : p.earlier_table) + (size_t)seq * p.width;
        for (int which = 0; which < 2; ++which, ++n) {
          const int s = n % NSLOT;
          if (n >= NSLOT && !mbar_wait(&kv_empty[s], ((n / NSLOT) - 1) & 1, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&kv_full[s], KV_BYTES);
          for (int pg = 0; pg < BKV / PAGE; ++pg) {
            int page = blk0 + pg < p.width ? pages[blk0 + pg] : -1;
            if (page < 0 || page >= p.n_pages) page = p.n_pages;       // a page that the step does not have: beyond the tensor, zeros
            const int row = (page * p.n_kv_heads + kvh) * PAGE;
            for (int h = 0; h < HALVES; ++h)
              tma_load_2d(ring + s * KV_BYTES + h * HALF_BYTES + pg * (PAGE * 128), which ? &map_v : &map_k,
                          &kv_full[s], h * 64, row);
          }
        }
      }
    }
  } else if (warp == kSoftmaxWarps + 1) {
    // ---- MMA issuer.  Two query tiles share every key and value tile.  Per key tile kt:
    //          O_A += P_A V(kt);  S_A = Q_A K(kt+1)^T;   O_B += P_B V(kt);  S_B = Q_B K(kt+1)^T
    //      so that while the softmax threads of one query tile work on its S, the tensor pipe runs the other
    //      tile's products.  P is written over the S it came from (as bf16, the first 64 columns) and is the
    //      A operand of P V from tensor memory; the next Q K^T of the same query tile is issued after that
    //      P V and the pipe runs in issue order, so it cannot overwrite a P that is still being read.  What is still to be waited
    //      for once P is there would leave the pipe idle between the two: the tiles are waited for before.
    //      The whole warp runs the loop (uniform values stay on the uniform datapath); only the tcgen05
    //      instructions sit under the elected lane. ----
    constexpr uint32_t idesc_s = instr_desc(BQ, BKV, 0);
    constexpr uint32_t idesc_o = instr_desc(BQ, D, 1);
    constexpr uint64_t kSlotUnits = KV_BYTES >> 4;      // a ring slot further, in the descriptor's 16-byte units
    const uint64_t dq[2] = {smem_desc(smem_u32(q_s), 16, 1024), smem_desc(smem_u32(q_s + Q_BYTES), 16, 1024)};
    const uint64_t dk0 = smem_desc(smem_u32(ring), 16, 1024), dv0 = smem_desc(smem_u32(ring), HALF_BYTES, 1024);
    int ks = 0, kph = 0, vs = 1, vph = 0, pph[2] = {0, 0}, first_pv[2] = {1, 1};      // ring slots and phases of the next K and V
    auto qk = [&](int x) {                              // (the elected lane) S_x = Q_x K^T on the key tile in slot ks
      const uint64_t dk = dk0 + (uint64_t)ks * kSlotUnits;
      umma_bf16_c<false>(tmem_s + x * 128, dq[x], dk, idesc_s);
#pragma unroll
      for (int k = 1; k < D / 16; ++k) {
        const uint64_t off = (uint64_t)(((k >> 2) * HALF_BYTES + (k & 3) * 32) >> 4);
        umma_bf16_c<true>(tmem_s + x * 128, dq[x] + off, dk + off, idesc_s);
      }
      umma_commit(&s_full[x]);
    };
    auto pv = [&](int x) {                              // (the elected lane) O_x += P_x V on the value tile in slot vs
      const uint64_t dv = dv0 + (uint64_t)vs * kSlotUnits;
      const uint32_t pa = tmem_s + x * 128, od = tmem_o + x * 128;
      if (first_pv[x]) umma_bf16_a_tmem_c<false>(od, pa, dv, idesc_o);
      else umma_bf16_a_tmem_c<true>(od, pa, dv, idesc_o);
#pragma unroll
      for (int j = 1; j < BKV / 16; ++j) umma_bf16_a_tmem_c<true>(od, pa + j * 8, dv + (uint64_t)(j * (2048 >> 4)), idesc_o);
    };
    auto landed = [&](uint64_t* bar, int parity) { return __all_sync(0xffffffffu, wait_soon(bar, parity, abort_flag)); };
    auto further = [&](int& s, int& ph) { s += 2; if (s >= NSLOT) { s -= NSLOT; ph ^= 1; } };
    // Which query tiles meet key tile kt (A a prefix of the axis, B a suffix; a share of it may have nothing for one of them).
    const int kb_b = has_b && kb_x[1] < ke_x[1] ? kb_x[1] : 0x7fffffff, ke_a = ke_x[0];
    ok = landed(&q_full, 0);
    if (kt0 < kt1) ok = ok && landed(&kv_full[ks], kph);
    if (ok && kt0 < kt1) {
      fence_after_sync();
      if (elect_one()) {
        if (ke_a > kt0) qk(0);
        if (kb_b == kt0) qk(1);
        umma_commit(&kv_empty[ks]);
      }
      __syncwarp();
      further(ks, kph);
    }
    for (int kt = kt0; kt < kt1 && ok; ++kt) {
      const bool a_now = kt < ke_a, b_now = kt >= kb_b, last = kt + 1 == kt1;
      const bool a_next = kt + 1 < ke_a, b_next = kt + 1 >= kb_b && !last;
      ok = landed(&kv_full[vs], vph) && (last || landed(&kv_full[ks], kph));
      if (ok && a_now) {
        ok = landed(&p_full[0], pph[0]);
        pph[0] ^= 1;
        fence_after_sync();
        if (ok && elect_one()) {
          pv(0);
          if (!b_now) umma_commit(&kv_empty[vs]);
          if (a_next) {
            qk(0);
            if (!b_next) umma_commit(&kv_empty[ks]);
          }
        }
        __syncwarp();
        first_pv[0] = 0;
      }
      if (ok && (b_now || b_next)) {
        if (b_now) {
          ok = landed(&p_full[1], pph[1]);
          pph[1] ^= 1;
        }
        fence_after_sync();
        if (ok && elect_one()) {
          if (b_now) {
            pv(1);
            umma_commit(&kv_empty[vs]);
          }
          if (b_next) {
            qk(1);
            umma_commit(&kv_empty[ks]);
          }
        }
        __syncwarp();
        if (b_now) first_pv[1] = 0;
      }
      further(ks, kph);
      further(vs, vph);
    }
    // every product has been issued: one arrival says that O of both query tiles is complete
    if (ok && elect_one()) { umma_commit(&o_done[0]); umma_commit(&o_done[1]); }
    __syncwarp();
  } else {
    // ---- softmax: warps 0-3 own query tile A, warps 4-7 tile B; thread r of a group owns query row r and all
    //      128 key columns of a tile (a warp may touch the 32 lanes of tensor memory given by its number modulo
    //      4).  Row maxima and sums need no shuffles.  O stays in tensor memory and is rescaled only when a row maximum has
    //      outgrown its reference. ----
    const int x = warp >> 2, row = tid & 127;
    const bool live = row < rows_x[x];
    const int qp = live ? p0_x[x] + row : -1;
    const int lo = live ? window_low(p.window_kind, p.window_size, qp) : 0;
    const int lo_last = window_low(p.window_kind, p.window_size, p1_x[x]);
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_row = tmem_s + x * 128 + lane_addr, o_row = tmem_o + x * 128 + lane_addr;
    float m_ref = -1e30f, l_run = 0.f;                  // reference maximum of the exponentials; the row's sum
    // > 0: the maximum may be taken before scaling.  Under a soft cap c a raw score s first becomes tanh(s scale / c)
    // (monotonic too) and the factor is c log2(e)
    const float sc = CAPPED ? p.cap_out : p.scale_log2, cap_in = p.cap_in;
    const int edge = live ? qp / PAGE * PAGE : 0;       // the row's own block begins here
    const int edge_first = p0_x[x] / PAGE * PAGE;
    int j = 0;
    bool okl = rows_x[x] > 0;
    for (int kt = kb_x[x]; kt < ke_x[x] && okl; ++kt, ++j) {
      const int key0 = key_tile(kt) * BKV;
      const bool exact = is_exact(kt);
      // (tensor-memory loads and votes are warp-wide: a warp gives up as a whole)
      okl = __all_sync(0xffffffffu, wait_soon(&s_full[x], j & 1, abort_flag));
      if (!okl) break;
      fence_after_sync();
      // a tile that lies wholly inside every row's window, and before every row's block, needs no position tests
      const bool no_mask = !exact && key0 + BKV <= edge_first && (key0 >= lo_last || key0 + BKV - 1 < keep);
      auto sees = [&](int first) {
        const int n = edge - first;
        const uint32_t before = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
        return visible(qp, lo, keep, first) & (exact ? ~before : before);
      };
      bool stored = false;
      if (!CAPPED && no_mask) {
        uint32_t r[BKV / 32][32];
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c) tmem_ld32_issue(s_row + c * 32, r[c]);
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c) landed32(r[c]);
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c)
#pragma unroll
          for (int g = 0; g < 16; ++g) mx4[g & 3] = max3(mx4[g & 3], __uint_as_float(r[c][2 * g]), __uint_as_float(r[c][2 * g + 1]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc;
        if (j == 0) m_ref = fmaxf(mx, m_ref);
        stored = !__any_sync(0xffffffffu, mx > m_ref + (m_ref < -1e29f ? 0.f : kWideSlack));
        if (stored) {
          const uint64_t sc2 = pair(sc, sc), nref2 = pair(-m_ref, -m_ref);
          uint64_t sum2[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < BKV / 32; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int g = 0; g < 16; ++g) {
              const float2 z = unpair(fma2(pair(__uint_as_float(r[c][2 * g]), __uint_as_float(r[c][2 * g + 1])), sc2, nref2));
              const float e0 = exp2_fast(z.x), e1 = exp2_fast(z.y);
              sum2[g & 1] = add2(sum2[g & 1], pair(e0, e1));
              w[g] = pack_bf16(e0, e1);
            }
            tmem_st16_nowait(s_row + c * 16, w);
          }
          const float2 sum = unpair(add2(sum2[0], sum2[1]));
          l_run += sum.x + sum.y;
        }
      }
      if (!stored) {
        auto seen = [&](int c) { return no_mask ? 0xffffffffu : sees(key0 + c * 32); };      // of columns 32 c .. 32 c + 31 by this row
        uint32_t some = 0, any = 0;                        // bit c: some row of the warp sees some of chunk c; columns that this row sees
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c) {
          const uint32_t in = seen(c);
          any |= in;
          some |= __any_sync(0xffffffffu, in != 0) ? 1u << c : 0u;
        }
        if (__any_sync(0xffffffffu, m_ref < -1e29f && any)) {
          // rows that have seen nothing so far (of their O and sum there is nothing to rescale)
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < BKV / 32; ++c) {
            if (!(some >> c & 1u)) continue;
            const uint32_t in = seen(c);
            uint32_t r[32];
            tmem_ld32_issue(s_row + c * 32, r);
            landed32(r);
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], (in >> e) & 1u ? __uint_as_float(r[e]) : -INFINITY);
            mx = fmaxf(mx, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
          }
          mx = CAPPED && mx > -INFINITY ? tanh_fast(mx * cap_in) * sc : mx * sc;
          if (m_ref < -1e29f) m_ref = fmaxf(mx, m_ref);
        }
        const uint64_t sc2 = pair(sc, sc);
        uint64_t sum2[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
        auto chunk = [&](int c, uint32_t (&r)[32]) {       // scores in r -> P, stored over columns of S that have been read
          uint32_t w[16];
          if (some >> c & 1u) {
            if (CAPPED || !no_mask) {
              const uint32_t in = seen(c);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                float v = __uint_as_float(r[e]);
                if (CAPPED) v = tanh_fast(v * cap_in);
                r[e] = (in >> e) & 1u ? __float_as_uint(v) : 0xff800000u;
              }
            }
            while (true) {
              const uint64_t nref2 = pair(-m_ref, -m_ref);
              uint64_t part[2] = {sum2[0], sum2[1]};
              float mx2[2] = {-INFINITY, -INFINITY};
#pragma unroll
              for (int g = 0; g < 16; ++g) {
                const float a = __uint_as_float(r[2 * g]), b = __uint_as_float(r[2 * g + 1]);
                mx2[g & 1] = max3(mx2[g & 1], a, b);
                const float2 z = unpair(fma2(pair(a, b), sc2, nref2));
                const float e0 = exp2_fast(z.x), e1 = exp2_fast(z.y);
                part[g & 1] = add2(part[g & 1], pair(e0, e1));
                w[g] = pack_bf16(e0, e1);
              }
              const float mx = fmaxf(mx2[0], mx2[1]) * sc;
              const bool grow = mx > m_ref + kWideSlack;
              if (!__any_sync(0xffffffffu, grow)) {
                sum2[0] = part[0];
                sum2[1] = part[1];
                break;
              }
              // A row's maximum has outgrown its reference, which is raised by a whole number: the factor is a power of two, so P that
              // has been rounded is not rounded again.  Every P V issued so far for this query tile has landed: the Q K^T whose S
              // was waited for above was issued after the last of them, and its arrival covers everything issued before it.
              const float m_new = grow ? fmaxf(m_ref + ceilf(mx - m_ref), mx) : m_ref, f = exp2f(m_ref - m_new);
              tmem_wait_st();
#pragma unroll 1
              for (int at = 0; at < D; at += 16) {
                uint32_t v[16];
                tmem_ld16(o_row + at, v);
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                tmem_st16_nowait(o_row + at, v);
              }
#pragma unroll 1
              for (int at = 0; at < c; ++at) {              // this tile's P so far
                uint32_t v[16];
                tmem_ld16(s_row + at * 16, v);
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = pack_bf16(__uint_as_float(v[e] << 16) * f, __uint_as_float(v[e] & 0xffff0000u) * f);
                tmem_st16_nowait(s_row + at * 16, v);
              }
              l_run *= f;
              const float2 s0 = unpair(sum2[0]), s1 = unpair(sum2[1]);
              sum2[0] = pair(s0.x * f, s0.y * f);
              sum2[1] = pair(s1.x * f, s1.y * f);
              m_ref = m_new;
            }
          } else {
#pragma unroll
            for (int g = 0; g < 16; ++g) w[g] = 0;
          }
          tmem_st16_nowait(s_row + c * 16, w);
        };
        uint32_t ra[32], rb[32];
        tmem_ld32_issue(s_row, ra);
        landed32(ra);
#pragma unroll 1
        for (int c = 0; c < BKV / 32; c += 2) {
          tmem_ld32_issue(s_row + (c + 1) * 32, rb);
          chunk(c, ra);
          landed32(rb);
          if (c + 2 < BKV / 32) tmem_ld32_issue(s_row + (c + 2) * 32, ra);
          chunk(c + 1, rb);
          if (c + 2 < BKV / 32) landed32(ra);
        }
        const float2 sum = unpair(add2(sum2[0], sum2[1]));
        l_run += sum.x + sum.y;
      }
      tmem_wait_st();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[x]);            // one arrival per warp
    }
    // the output: O / l once the last P V is done
    ok = okl && !abort_s && j > 0;
    const size_t at = (size_t)(tok0 + x * BQ + row) * p.n_heads + head;
    if (p.n_splits > 1 && live) {
      // what this share adds up to: the row's sum and what it is measured against (nothing: a sum of zero)
      p.part_ml[at * p.n_splits + blockIdx.z] = make_float2(m_ref, j > 0 ? l_run : 0.f);
    }
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&o_done[x], 0, abort_flag));
    fence_after_sync();
    if (ok) {
      // A thread has a row, a line of 128 bytes at a time; through shared memory (that of the queries, which are done with) the lines
      // go out whole: 8 lanes to each.
      uint8_t* mine = q_s + warp * 4096;
      const size_t row0 = (size_t)(tok0 + x * BQ + (warp & 3) * 32) * p.n_heads + head;
      const int n_rows = rows_x[x] - (warp & 3) * 32;     // of this warp (may be none)
      // a sink adds 2^(sink log2 e - reference) to the row's sum and nothing to O; the exponent is capped so that a
      // sink far above every score gives a huge finite sum
      if (p.sink && p.n_splits == 1) l_run += exp2f(fminf(p.sink[head] * 1.4426950408889634f - m_ref, 120.f));
      const float inv = 1.0f / fmaxf(l_run, 1e-20f);
      auto put = [&](int chunk, uint4 v) { *reinterpret_cast<uint4*>(mine + lane * 128 + ((chunk ^ (lane & 7)) << 4)) = v; };
      auto lines = [&](uint8_t* to, size_t stride) {      // the warp's 32 lines to memory, `stride` bytes apart
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (lane >> 3), chunk = lane & 7;
          const uint4 v = *reinterpret_cast<const uint4*>(mine + r * 128 + ((chunk ^ (r & 7)) << 4));
          if (r < n_rows) *reinterpret_cast<uint4*>(to + r * stride + chunk * 16) = v;
        }
        __syncwarp();
      };
      if (p.n_splits > 1) {
        uint8_t* to = reinterpret_cast<uint8_t*>(p.part_o + (row0 * p.n_splits + blockIdx.z) * D);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float v[32];
          tmem_ld32(o_row + c, v);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            put(e, make_uint4(__float_as_uint(v[4 * e]), __float_as_uint(v[4 * e + 1]), __float_as_uint(v[4 * e + 2]), __float_as_uint(v[4 * e + 3])));
          lines(to + c * 4, (size_t)p.n_heads * p.n_splits * D * 4);
        }
      } else {
        uint8_t* to = reinterpret_cast<uint8_t*>(p.out + row0 * D);
#pragma unroll 1
        for (int c = 0; c < D; c += 64) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float v[32];
            tmem_ld32(o_row + c + half * 32, v);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              put(half * 4 + e, make_uint4(pack_bf16(v[8 * e] * inv, v[8 * e + 1] * inv), pack_bf16(v[8 * e + 2] * inv, v[8 * e + 3] * inv),
                                           pack_bf16(v[8 * e + 4] * inv, v[8 * e + 5] * inv), pack_bf16(v[8 * e + 6] * inv, v[8 * e + 7] * inv)));
          }
          lines(to + c * 2, (size_t)p.n_heads * D * 2);
        }
      }
    }
    fence_before_sync();
  }
  if (abort_s) {
    if (tid == 0 && p.error_flag) atomicExch(p.error_flag, 2);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base_s), "r"(TMEM_COLS));
}

// The shares of a query tile's keys joined: out[t, h] = sum_s w_s O_s / (sum_s w_s l_s + sink), w_s = 2^(m_s - max m).  A warp per
// (token, head), four features or two per lane.
template <int D>
__global__ void __launch_bounds__(256) attention_prefill_combine(const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                                                                 __nv_bfloat16* __restrict__ out, long rows, int n_splits,
                                                                 const float* __restrict__ sink, int n_heads) {
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  const long th = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_launch_dependents();
  if (th >= rows) return;
  const float2 ml = lane < n_splits ? __ldcg(part_ml + th * n_splits + lane) : make_float2(-1e30f, 0.f);
  const float M = warp_max(ml.x);
  const float w = exp2f(ml.x - M), l = ml.y > 0.f || ml.y != ml.y ? w * ml.y : 0.f;
  float L = warp_sum(l), acc[PER] = {};
  for (int s = 0; s < n_splits; ++s) {
    const float ws = __shfl_sync(0xffffffffu, w, s), ls = __shfl_sync(0xffffffffu, ml.y, s);
    if (ls == 0.f) continue;                             // (this share held nothing for the row, or was not written)
    const float* src = part_o + (th * n_splits + s) * D + lane * PER;
    if (PER == 4) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
      acc[0] += ws * v.x; acc[1] += ws * v.y; acc[PER - 2] += ws * v.z; acc[PER - 1] += ws * v.w;
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
      acc[0] += ws * v.x; acc[1] += ws * v.y;
    }
  }
  if (sink) L += exp2f(fminf(sink[th % n_heads] * 1.4426950408889634f - M, 120.f));
  const float inv = 1.0f / fmaxf(L, 1e-20f);
  uint32_t* dst = reinterpret_cast<uint32_t*>(out + th * D + lane * PER);
#pragma unroll
  for (int i = 0; i < PER / 2; ++i) dst[i] = pack_bf16(acc[2 * i] * inv, acc[2 * i + 1] * inv);
}

}  // namespace pre8
}  // namespace cpi

using namespace cpi;

// q, out [T, NH*D] bfloat16; k_pages, v_pages [n_pages, NKV, 64, D] bfloat16, named per sequence of the
// step and block by earlier_table and exact_table [sequences, width] (-1: none).  `n_splits` > 1: that many blocks of threads share a query tile's
// keys, through `scratch` (n_tokens * n_heads * n_splits * (head_dim + 2) floats).
extern "C" int cpi_attention_prefill_kv8(const void* q, void* out, const void* k_pages, const void* v_pages, long n_pages,
                                         const int* earlier_table, const int* exact_table, int n_seqs, int width, const int* token_seq,
                                         const int* token_pos, const int* tile_tok0, const int* tile_rows, int n_tiles, int n_tokens,
                                         int n_heads, int n_kv_heads, int head_dim, int window_kind, int window_size, int keep_first,
                                         float scale, float softcap, const float* sink, int n_splits, float* scratch, int* error_flag,
                                         cudaStream_t stream) {
  if (n_tiles == 0 || n_tokens == 0) return 0;
  const long rows = (long)n_tokens * n_heads;
  CPI_REQUIRE(n_splits >= 1 && n_splits <= 32 && (n_splits == 1 || scratch), "attention_prefill_kv8: %d shares (up to 32, with scratch)", n_splits);
  CPI_REQUIRE(n_kv_heads >= 1 && n_heads % n_kv_heads == 0 && (head_dim == 64 || head_dim == 128),
              "attention_prefill_kv8: unsupported shape (heads %d/%d, head size %d)", n_heads, n_kv_heads, head_dim);
  CPI_REQUIRE(window_kind == 0 || window_size > 0, "attention_prefill_kv8: window kind %d needs a size > 0", window_kind);
  CPI_REQUIRE(n_tiles <= 65535, "attention_prefill_kv8: too many query tiles in one launch (%d)", n_tiles);
  const uint64_t kv_rows = (uint64_t)n_pages * n_kv_heads * pre8::PAGE;
  CPI_REQUIRE(n_pages > 0 && kv_rows + (uint64_t)n_kv_heads * pre8::PAGE < (1ull << 31), "attention_prefill_kv8: %ld pages of %d heads", n_pages, n_kv_heads);
  CUtensorMap mq, mk, mv;
  const uint64_t q_width = (uint64_t)n_heads * head_dim;
  if (tc::get_map_2d_bf16(q, q_width, (uint64_t)n_tokens, q_width * 2, 64, pre::BQ, &mq)) return 1;
  if (tc::get_map_2d_bf16(k_pages, (uint64_t)head_dim, kv_rows, (uint64_t)head_dim * 2, 64, pre8::PAGE, &mk)) return 1;
  if (tc::get_map_2d_bf16(v_pages, (uint64_t)head_dim, kv_rows, (uint64_t)head_dim * 2, 64, pre8::PAGE, &mv)) return 1;
  pre8::Params p{(__nv_bfloat16*)out, earlier_table, exact_table, width, token_pos, token_seq, tile_tok0, tile_rows,
                n_heads, n_kv_heads, window_kind, window_size, keep_first > 0 ? keep_first : 0, scale * 1.4426950408889634f, error_flag, sink,
                softcap > 0.f ? scale / softcap : 0.f, softcap > 0.f ? softcap * 1.4426950408889634f : 0.f, (int)n_pages, n_tokens, n_seqs, n_splits, scratch,
                scratch ? reinterpret_cast<float2*>(scratch + rows * n_splits * head_dim) : nullptr};
  dim3 grid(n_heads, n_tiles, n_splits);
  // One block of threads to an SM: each takes all of the tensor memory.  Two heads' worth of 64 would fit an SM's shared memory, and
  // a second block that is put there, while the kernel before still fills the other SMs, waits for the first to end (four windowed
  // prompts, 144 blocks: 80 us instead of 47).
  const int smem = head_dim == 64 ? 120 * 1024 : head_dim / 64 * 128 * 128 * (2 + pre8::kRingSlots);
  auto launch = [&](auto dim, auto capped) {
    auto* kernel = pre8::attention_prefill_kv8_kernel<dim.value, capped.value>;
    static bool set[64] = {};                              // per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || !set[dev]) {
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (dev >= 0 && dev < 64) set[dev] = true;
    }
    cpi::launch_pdl(kernel, grid, pre8::kThreads, smem, stream, mq, mk, mv, p);
  };
  auto launch_dim = [&](auto dim) {
    if (p.cap_out > 0.f) launch(dim, std::true_type{}); else launch(dim, std::false_type{});
  };
  if (head_dim == 128) launch_dim(std::integral_constant<int, 128>{}); else launch_dim(std::integral_constant<int, 64>{});
  if (check_launch("attention_prefill_kv8")) return 2;
  if (n_splits == 1) return 0;
  auto* combine = head_dim == 128 ? pre8::attention_prefill_combine<128> : pre8::attention_prefill_combine<64>;
  cpi::launch_pdl(combine, dim3((unsigned)((rows + 7) / 8)), 256, 0, stream, p.part_o, p.part_ml, p.out, rows, n_splits, sink, n_heads);
  return check_launch("attention_prefill_combine");
}
CPI_PACKED(cpi_attention_prefill_kv8)
