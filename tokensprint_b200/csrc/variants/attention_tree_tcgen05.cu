// Attention of a tree of drafted tokens over the paged cache on the 5th-generation tensor cores: bfloat16, heads of 64 and 128.
//
// What it computes stands in attention_tree.cu.  A group of up to two tiles of 128 (node, query head) rows walks the keys of its request and KV head in blocks of
// 128: S = Q K^T and O += P V by tcgen05.mma with S, P and O in tensor memory, K and V brought page by page by TMA into rings.
//
// What bounds a step is reading the cache: 64 KB a block at 44 GB/s an SM are 1.5 us, the products of one tile 0.55.  The rest follows from that:
// * Persistent CTAs, each with an even share of all (request, KV head, group, block)s, worked out on the device: lengths and trees differ, and a
//   captured step serves them all.  A group whose blocks fall to several CTAs leaves parts, joined by a second kernel in a fixed order.
// * The copying warps run ahead over the ends of groups, so that the rings stay full while a group's results leave.
// * Groups of one tile take turns on two accumulators: tile 0 the even blocks, tile 1 the odd ones, so that one block's exponentials run beside the next one's products.
// * Few rows would leave the exponentials of a block to one warp: up to 64 rows stand in the tile twice, up to 32 four times, and every copy weighs its own
//   half or quarter of the block's keys (the others' weights are zero).  The copies' sums are added when the group is done.
//
// A row's maximum is raised only when it lags more than 2^8 behind (the weights stay far inside bfloat16's range, and the division by the sum, taken with
// the same maximum, cancels it).  Weights are rounded to bfloat16 for the product with the values, their own type; sums take them unrounded.
// Every wait is bounded: one that gives up raises the error word, and the CTA ends in order.
//
// Times below of 4 trees of 61 at 30,000 rows are of short bursts at 1.95 GHz, where the present kernel takes 218 us; in a loop of seconds the power cap holds 1.5 GHz, and it
// takes 260.
#include <math.h>

#include "../common.cuh"
#include "kv_tensor_map.cuh"

#if TS_HEAD_DIM != 64 && TS_HEAD_DIM != 128
#error "attention_tree_tcgen05.cu is written for heads of 64 and 128"
#endif

namespace {

constexpr int D = TS_HEAD_DIM;
constexpr int BM = 128, BN = 128;
constexpr int HALVES = D / 64;
constexpr uint32_t ATOM = 128 * 128;             // [128 rows x 128 bytes]: 64 entries of every row, swizzled
constexpr uint32_t TILE = HALVES * ATOM;         // Q of a tile, K or V of a block
constexpr int CH = 16;                           // columns of the result that pass from the lanes that hold them to whole lines at a time
constexpr uint32_t MERGE = 8 * 32 * CH * 4;       // a half of the columns each for two times four warps
constexpr int MAX_NODES = 256;
constexpr int THREADS = 384;                     // eight warps of softmax, three that copy (the last also plans), one that issues products
constexpr int AHEAD = 4;                         // pieces of work that are planned ahead
constexpr uint32_t SPIN_LIMIT = 1u << 22;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LAG = 8.f;
// What a block costs, in parts of a group of one tile's: shares are even in this measure.
constexpr int COST_ONE = 1, COST_TWO = 2;

// Builds of the kernel: WIDE, for groups of up to two tiles of rows, else of one (K has a third stage where the second tile's Q would lie).
template <bool WIDE>
struct Layout {
  static constexpr int NK = D == 64 ? 4 : WIDE ? 2 : 3, NV = D == 64 ? 4 : 2;
  static constexpr uint32_t Q = 0, MERGE_AT = (WIDE ? 2 : 1) * TILE, K = MERGE_AT + MERGE, V = K + NK * TILE, BYTES = V + NV * TILE;
};
static_assert(Layout<true>::BYTES <= 216 * 1024 && Layout<false>::BYTES <= 216 * 1024, "beside it 1 KB to align and 7 KB of plans");

struct Params {
  __nv_bfloat16* out;     // [T, nq, D]
  const unsigned long long* mask;  // [T, words]
  const int* cu;          // [B + 1]
  const int* context;     // [B]
  const int* table;       // [B, max_blocks]
  const int* positions;   // [T] or null
  const float* head_sinks;  // [nq] or null
  float* part_o;          // [CTA, 2, part_rows, D]
  float* part_ml;         // [CTA, 2, part_rows, 2]
  int4* plan;             // [CTA, 2] the group of rows whose first part is this CTA's, for the joining kernel: (first token, row, rows, KV head), (last CTA or 0, slot, -, -)
  int* error;
  int words, max_blocks, page, nq, nkv, window, num_seqs, total_slots, part_rows, ctas;
  float scale_log2, cap_log2, cap_inv;  // cap * log2(e) and scale / cap
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1  // (the waits are many: unrolled they alone overflow the instruction cache)
  for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if (*abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
// K-major operand, 128-byte swizzle: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// MN-major operand (V as [key][dim]): rows of 64 dims, 8-key groups 1024 bytes apart, the second 64 dims ATOM bytes further.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((ATOM >> 4) & 0x3FFF) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// D = A B and D += A B, A and B in shared memory
__device__ __forceinline__ void umma_first(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 0, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
}
__device__ __forceinline__ void umma_more(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
}
// the same with A (P, [128 rows x 16 keys], two bfloat16 per column) in tensor memory
__device__ __forceinline__ void umma_tmem_a(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool more) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)more) : "memory");
}
__device__ __forceinline__ void umma_tmem_a_more(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(chosen));
  return chosen != 0;
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// float32 accumulators, bfloat16 operands, A K-major; B K-major or MN-major
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}

// ---------------------------------------------------------------------------
// who does what

// A request as the plan sees it: its key blocks kb0 .. kb0 + blocks - 1, its rows for a KV head and their groups.
struct Request {
  int q_begin, t, n, kb0, blocks, rows, groups;
  int whole_from;  // the row from which on a window hides nothing of what is before the step
};
template <bool WIDE>
__device__ __noinline__ Request request_of(const Params& p, int b, int RT) {
  Request r;
  r.q_begin = p.cu[b];
  r.t = p.cu[b + 1] - r.q_begin;
  r.n = p.context[b];
  r.rows = r.t > 0 ? r.t * (p.nq / p.nkv) : 0;
  r.groups = (r.rows + (WIDE ? 2 * RT : RT) - 1) / (WIDE ? 2 * RT : RT);
  int lo = 0;
  r.whole_from = 0;
  if (p.window > 0 && r.t > 0) {  // the first row that any node sees
    int lowest = INT_MAX, highest = 0;
#pragma unroll 1
    for (int i = 0; i < r.t; i += 8) {  // (eight loads on their way: one behind the other they take 600 cycles each)
      int x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = p.positions[r.q_begin + min(i + j, r.t - 1)];
#pragma unroll
      for (int j = 0; j < 8; ++j) lowest = min(lowest, x[j]), highest = max(highest, x[j]);
    }
    r.whole_from = max(highest - p.window + 1, 0);
    const long long from = (long long)lowest - p.window + 1;
    lo = from < 0 ? 0 : from > r.n - r.t ? max(r.n - r.t, 0) : (int)from;
  }
  r.kb0 = lo / BN;
  r.blocks = r.t > 0 && r.n > 0 ? (r.n - 1) / BN - r.kb0 + 1 : 0;
  if (r.t > 0 && r.blocks < 1) r.blocks = 1;  // nobody sees anything: zeros are written all the same
  return r;
}
// What a block of the request's group g costs.
template <bool WIDE>
__device__ __forceinline__ int cost_of(const Request& r, int g, int RT) {
  return WIDE && r.rows - g * 2 * RT > RT ? COST_TWO : COST_ONE;
}
template <bool WIDE>
__device__ __forceinline__ int cost_of_head(const Request& r, int RT) {  // of all its groups
  return r.groups == 0 ? 0 : r.blocks * ((r.groups - 1) * (WIDE ? COST_TWO : COST_ONE) + cost_of<WIDE>(r, r.groups - 1, RT));
}

// A piece of work: nb key blocks from kb on for the rows r0 .. r0 + rows - 1 of a request and KV head.
struct __align__(16) Piece {
  int b, hk, q_begin, t;
  int n, kb, nb, r0;  // nb 0: no more pieces
  int rows, sets, whole, slot;
  int last_cta, first_blk, whole_from, pad;   // where the group's last blocks fall; the group's block kb; see Request
};

// How the rows of a piece lie in the tensor memory: `sets` sets of 32 rows in different warps (8: two tiles of rows; 4, 2, 1: one tile once, twice, four times, in
// each of the two accumulators).  Warp w holds set w % sets.
__device__ __forceinline__ int sets_of(int rows_of_group, int RT) { return rows_of_group > RT ? 8 : rows_of_group > 64 ? 4 : rows_of_group > 32 ? 2 : 1; }

// Walks over the pieces of one CTA's share [from, to); the lanes of a warp walk together.
template <bool WIDE>
struct Walk {
  int b, hk, g, from, to, at, share;  // at: where group (b, hk, g) begins
  Request r;
  // The batch is added up by every warp for itself, 32 requests at a time: no memory, no barrier between.
  __device__ __forceinline__ void begin(const Params& p, int RT) {
    const int lane = threadIdx.x & 31;
    int total = 0;
    Request mine;
    int cost = 0, sum = 0;
    auto scan = [&](int b0) {
      cost = 0;
      if (b0 + lane < p.num_seqs) {
        mine = request_of<WIDE>(p, b0 + lane, RT);
        cost = cost_of_head<WIDE>(mine, RT) * p.nkv;
      }
      sum = cost;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
    };
#pragma unroll 1
    for (int b0 = 0; b0 < p.num_seqs; b0 += 32) {
      scan(b0);
      total += __shfl_sync(0xffffffffu, sum, 31);
    }
    share = max(COST_TWO, (total + p.ctas - 1) / p.ctas);  // (at least a block: every CTA between a group's first and last has a part of it)
    from = (int)min((long long)blockIdx.x * share, (long long)total);
    to = (int)min((long long)from + share, (long long)total);
    b = p.num_seqs, hk = g = 0, at = total;
    r.groups = 0;
    if (from >= to) return;
    int before = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < p.num_seqs; b0 += 32) {
      if (p.num_seqs > 32) scan(b0);  // (else it is there still)
      const unsigned here = __ballot_sync(0xffffffffu, from >= before + sum - cost && from < before + sum);
      if (here != 0) {
        const int who = __ffs(here) - 1;
        r.q_begin = __shfl_sync(0xffffffffu, mine.q_begin, who);
        r.t = __shfl_sync(0xffffffffu, mine.t, who);
        r.n = __shfl_sync(0xffffffffu, mine.n, who);
        r.kb0 = __shfl_sync(0xffffffffu, mine.kb0, who);
        r.blocks = __shfl_sync(0xffffffffu, mine.blocks, who);
        r.rows = __shfl_sync(0xffffffffu, mine.rows, who);
        r.groups = __shfl_sync(0xffffffffu, mine.groups, who);
        r.whole_from = __shfl_sync(0xffffffffu, mine.whole_from, who);
        before += __shfl_sync(0xffffffffu, sum - cost, who);
        b = b0 + who;
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (b >= p.num_seqs) return;
    const int head = cost_of_head<WIDE>(r, RT), group = r.blocks * (WIDE ? COST_TWO : COST_ONE);
    hk = (from - before) / head;
    g = min((from - before - hk * head) / group, r.groups - 1);
    at = before + hk * head + g * group;
  }
  __device__ __forceinline__ bool next(const Params& p, int RT, Piece& out) {
#pragma unroll 1
    while (b < p.num_seqs && at < to) {
      if (r.groups == 0 || g >= r.groups) {
        g = 0;
        if (r.groups == 0 || ++hk >= p.nkv) {
          hk = 0;
          if (++b < p.num_seqs) r = request_of<WIDE>(p, b, RT);
          continue;
        }
      }
      const int cost = cost_of<WIDE>(r, g, RT);
      // blocks whose beginning lies in [from, to)
      const int blk0 = from > at ? (from - at + cost - 1) / cost : 0, blk1 = min(r.blocks, (to - at + cost - 1) / cost);
      const int RG = WIDE ? 2 * RT : RT, r0 = g * RG, rows = min(r.rows - r0, RG);
      // (a share has two groups in part at most, its first and its last: their places in scratch)
      out = Piece{b, hk, r.q_begin, r.t, r.n, r.kb0 + blk0, blk1 - blk0, r0, rows, sets_of(rows, RT), blk0 == 0 && blk1 == r.blocks, at <= from ? 0 : 1, (at + (r.blocks - 1) * cost) / share, blk0, r.whole_from, 0};
      at += r.blocks * cost;
      ++g;
      if (blk0 < blk1) return true;
    }
    out.nb = 0;
    return false;
  }
};

// Which of the 32 keys from `base` on a node sees, as bits.
__device__ __noinline__ uint32_t seen_bits(const Params& p, int q_begin, int t, int n, int token, int pos, int base) {
  const int first = n - t;
  uint32_t out = 0;
  const int ahead = first - base;  // keys of these 32 ahead of the step's rows
  if (ahead > 0) {
    out = ahead >= 32 ? 0xffffffffu : (1u << ahead) - 1;
    if (p.window > 0) {
      const long long hidden = (long long)pos - p.window + 1 - base;
      out = hidden >= 32 ? 0u : hidden > 0 ? out & ~((1u << (int)hidden) - 1) : out;
    }
  }
  if (ahead < 32 && base < n) {
    const unsigned long long* words = p.mask + (size_t)token * p.words;
    const int from = max(-ahead, 0);  // the first node among these keys
    const int w = from >> 6, off = from & 63;
    unsigned long long x = w < p.words ? words[w] >> off : 0ull;
    if (off > 32 && w + 1 < p.words) x |= words[w + 1] << (64 - off);
    uint32_t bits = (uint32_t)x;
    const int nodes = min(t - from, 32);
    bits = nodes >= 32 ? bits : nodes > 0 ? bits & ((1u << nodes) - 1) : 0u;
    if (p.window > 0) {
      for (uint32_t left = bits; left != 0; left &= left - 1) {
        const int i = __ffs(left) - 1;
        if (p.positions[q_begin + from + i] <= pos - p.window) bits &= ~(1u << i);
      }
    }
    out |= ahead > 0 ? bits << ahead : bits;
  }
  return out;
}

// 32 scores of a row: -inf for keys that its node does not see.
__device__ __forceinline__ void hide(uint32_t bits, uint32_t (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!((bits >> i) & 1)) v[i] = 0xff800000u;
}
__device__ __forceinline__ float largest(const uint32_t (&v)[32]) {
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(v[i]));
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
// two float32 in one 64-bit register, and the packed arithmetic on them
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 32 scores to 16 pairs of weights; returns their sum.  (With every fourth or second pair's exponentials on the FMA units instead of the special-function one:
// 4 trees of 61 at 30,000 rows 222 -> 231, 258 us; what the weights wait for is tensor memory.)
__device__ __forceinline__ float weights(const uint32_t (&v)[32], uint32_t (&w)[16], float scale, float off) {
  const uint64_t scale2 = pack2(scale, scale), off2 = pack2(-off, -off);
  uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t x = fma2(pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), scale2, off2);
    float a, b;
    unpack2(x, a, b);
    a = fast_exp2(a), b = fast_exp2(b);
    sum[i & 3] = add2(sum[i & 3], pack2(a, b));
    w[i] = pack_bf16(a, b);
  }
  float a, b;
  unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), a, b);
  return a + b;
}

// cap * tanh(x), in units of log2: tanh(x) = 1 - 2 / (exp(2x) + 1), exact at both ends, absolute error of a few 1e-7 in between.
__device__ __forceinline__ void bend(const Params& p, uint32_t (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(p.cap_log2 * (1.f - __fdividef(2.f, __expf(2.f * p.cap_inv * __uint_as_float(v[i])) + 1.f)));
}

// One block's weights for one warp's 32 rows: 32 N keys from column `key0` of the block on.  Scores come from `s_addr` (the tile's columns at this warp's lanes); the
// weights of all 128 keys go over them as bfloat16, zeros for keys that are other copies' part.  Of 128 keys the second 64 are kept between the look for the
// largest and the weights, and the first are read again: all would not fit the registers.
template <int N, bool CAP>
__device__ __forceinline__ void weigh(const Params& p, const Piece& r, int token, int pos, int kbase, int key0, bool open, uint32_t s_addr, uint32_t o_addr, bool first_item,
                                      float scale, float& m_run, float& l_run) {
  constexpr int H = N < 2 ? N : 2;  // 32s of keys that are held
  uint32_t v[H][32], bits[N];
  if (!open) {
#pragma unroll
    for (int c = 0; c < N; ++c) bits[c] = token >= 0 ? seen_bits(p, r.q_begin, r.t, r.n, token, pos, kbase + key0 + 32 * c) : 0u;
  }
  float m_blk = -INFINITY;
#pragma unroll
  for (int c0 = 0; c0 < N; c0 += H) {
#pragma unroll
    for (int h = 0; h < H; ++h) tmem_ld32(s_addr + key0 + 32 * (c0 + h), v[h]);
    tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (CAP) bend(p, v[h]);
      if (!open) hide(bits[c0 + h], v[h]);
      m_blk = fmaxf(m_blk, largest(v[h]));
    }
  }
  m_blk *= scale;                          // (scale > 0)
  const bool raise = m_blk - m_run > LAG;  // also where m_run is -inf and m_blk is not
  if (__any_sync(0xffffffffu, raise)) {
    const float m_new = raise ? m_blk : m_run;
    const float corr = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
    m_run = m_new;
    l_run *= corr;
    if (!first_item) {
      // (the product before this one on the accumulator is complete: the scores, asked for behind it, are)
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        uint32_t o[16];
        tmem_ld16(o_addr + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
        tmem_st16(o_addr + c, o);
      }
    }
  }
  const float off = m_run == -INFINITY ? 0.f : m_run;
  uint32_t w[H][16];
#pragma unroll
  for (int h = 0; h < H; ++h) l_run += weights(v[h], w[h], scale, off);
  if (N == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) tmem_ld32(s_addr + 32 * h, v[h]);
    tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // (the kept ones' place is over scores that have been read by now)
      tmem_st16(s_addr + 32 + 16 * h, w[h]);
      if (CAP) bend(p, v[h]);
      if (!open) hide(bits[h], v[h]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l_run += weights(v[h], w[h], scale, off);
      tmem_st16(s_addr + 16 * h, w[h]);
    }
  } else {
#pragma unroll
    for (int h = 0; h < H; ++h) tmem_st16(s_addr + key0 / 2 + 16 * h, w[h]);
#pragma unroll
    for (int i = 0; i < 16; ++i) w[0][i] = 0u;
#pragma unroll
    for (int c = 16 * N; c < 64; c += 16) tmem_st16(s_addr + (key0 / 2 ^ c), w[0]);  // (key0 is a multiple of 32 N: the other multiples of 16)
  }
  tmem_st_wait();
}

// A finished piece's rows leave: whole groups as results, others as parts.
// Warp (half, quad) takes half of the columns of both accumulators at its 32 lanes.  Rows that stand there once leave from the registers; copies in
// other lanes are added up through shared memory, CH columns at a time.  Parts stand as [4 columns][row][4], so that lanes write and read whole lines.
template <int SETS>
__device__ __noinline__ void leave(const Params& p, const Piece& w, bool good, int G, int RT, const float2 (*ml)[32], unsigned char* merge, uint32_t tmem, int warp, int lane) {
  constexpr int TILES = SETS == 8 ? 2 : 1;  // of rows; else the two accumulators hold the same rows
  const int half = warp >> 2, quad = warp & 3, c_begin = half * (D / 2);
  const uint32_t o_lane = tmem + ((uint32_t)(quad * 32) << 16) + 256 + c_begin;
  const size_t part = ((size_t)blockIdx.x * 2 + w.slot) * p.part_rows;
  const bool both = w.nb > 1;  // the second accumulator holds something too
#pragma unroll
  for (int x = 0; x < TILES; ++x) {
    const int in = (SETS == 8 ? quad : quad % SETS) * 32 + lane, place = x * BM + in, row = w.r0 + x * RT + in;
    const bool real = in < RT && x * RT + in < w.rows, kept = good && place < p.part_rows;
    // the row's maximum and sum over its copies, and what this lane's sums are multiplied by
    float2 y[8 / SETS];
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8 / SETS; ++i) y[i] = ml[(place >> 5) + i * SETS][lane], top = fmaxf(top, y[i].x);
#pragma unroll
    for (int i = 0; i < 8 / SETS; ++i) sum += y[i].x == -INFINITY ? 0.f : y[i].y * fast_exp2(y[i].x - top);
    const float m0 = ml[(SETS == 8 ? 4 * x : 0) + quad][lane].x, m1 = ml[4 + quad][lane].x;
    float all = 1.f;
    if (w.whole) {
      float down = 1.f;
      if (p.head_sinks != nullptr && real) {
        const float sink = p.head_sinks[w.hk * G + row % G] * LOG2E, over = fmaxf(top, sink);
        down = top == -INFINITY ? 0.f : fast_exp2(top - over);
        sum = sum * down + (sink == -INFINITY ? 0.f : fast_exp2(sink - over));
      }
      all = sum > 0.f ? down / sum : 0.f;
    } else if (half == 0 && quad < SETS && kept) {
      *reinterpret_cast<float2*>(p.part_ml + (part + place) * 2) = make_float2(top, sum);
    }
    const float f0 = m0 == -INFINITY ? 0.f : all * fast_exp2(m0 - top), f1 = SETS == 8 || !both || m1 == -INFINITY ? 0.f : all * fast_exp2(m1 - top);
    __nv_bfloat16* out = p.out + ((size_t)(w.q_begin + row / G) * p.nq + w.hk * G + row % G) * D + c_begin;
    float* to_part = p.part_o + part * D + ((size_t)(c_begin / 4) * p.part_rows + place) * 4;
    const int step = p.part_rows * 4;
    unsigned char* mine = merge + half * (MERGE / 2) + (quad * 32 + lane) * (CH * 4);
    const int swizzle = (lane >> 1 & 3) << 4;
#pragma unroll 1
    for (int c = 0; c < D / 2; c += CH) {
      uint32_t o0[CH], o1[CH];
      tmem_ld16(o_lane + x * D + c, o0);
      if (SETS < 8 && both) tmem_ld16(o_lane + D + c, o1);
      tmem_ld_wait();
      float v[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        v[i] = f0 > 0.f ? __uint_as_float(o0[i]) * f0 : 0.f;
        if (SETS < 8 && f1 > 0.f) v[i] = fmaf(__uint_as_float(o1[i]), f1, v[i]);
      }
      // of a row's four pieces of 4 columns: which this warp adds up and writes (its copies' warps share them)
      constexpr int PIECES = SETS >= 4 ? 4 : SETS, COPIES = SETS >= 4 ? 1 : 4 / SETS;
      const int first = SETS >= 4 ? 0 : SETS == 2 ? (quad >> 1) * 2 : quad;
      if (SETS < 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(mine + ((i << 4) ^ swizzle)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
        const unsigned char* row_at = merge + half * (MERGE / 2) + ((quad % SETS) * 32 + lane) * (CH * 4);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          float4 z[COPIES];
#pragma unroll
          for (int k = 0; k < COPIES; ++k) z[k] = *reinterpret_cast<const float4*>(row_at + k * (SETS * 32 * CH * 4) + (((first + i) << 4) ^ swizzle));
#pragma unroll
          for (int k = 1; k < COPIES; ++k) z[0].x += z[k].x, z[0].y += z[k].y, z[0].z += z[k].z, z[0].w += z[k].w;
          v[4 * i] = z[0].x, v[4 * i + 1] = z[0].y, v[4 * i + 2] = z[0].z, v[4 * i + 3] = z[0].w;
        }
        asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
      }
      if (w.whole) {
        if (real && good) {
#pragma unroll
          for (int i = 0; i < PIECES; ++i)
            *reinterpret_cast<uint2*>(out + c + 4 * (first + i)) = make_uint2(pack_bf16(v[4 * i], v[4 * i + 1]), pack_bf16(v[4 * i + 2], v[4 * i + 3]));
        }
      } else if (kept) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
          *reinterpret_cast<float4*>(to_part + (size_t)(c / 4 + first + i) * step) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    }
  }
}

template <bool WIDE, bool CAP>
__global__ void __launch_bounds__(THREADS, 1) attention_tree_kernel(const __grid_constant__ CUtensorMap map_q1, const __grid_constant__ CUtensorMap map_q2,
                                                                    const __grid_constant__ CUtensorMap map_q4, const __grid_constant__ CUtensorMap map_k,
                                                                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Params params) {
  using L = Layout<WIDE>;
  constexpr int NK = L::NK, NV = L::NV;
  ts_pdl_wait();  // tensor memory is never held while waiting for another kernel
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t q_full, q_empty, k_full[NK], k_empty[NK], v_full[NV], v_empty[NV], s_full[2], p_full[2], o_full[2], piece_full[AHEAD], piece_empty[AHEAD], all_done;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;
  __shared__ float2 ml_s[8][32];
  __shared__ Piece piece_s[AHEAD];
  __shared__ Params params_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // The arguments in shared memory: what is read once a piece is seldom in the constant cache.
  static_assert(sizeof(Params) % 4 == 0 && sizeof(Params) / 4 <= THREADS, "a word per thread");
  if (tid < (int)(sizeof(Params) / 4)) reinterpret_cast<uint32_t*>(&params_s)[tid] = reinterpret_cast<const uint32_t*>(&params)[tid];
  __syncthreads();
  const Params& p = params_s;
  const int G = p.nq / p.nkv, RT = BM / G * G;

  if (warp == 9 && lane < 5)
    asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &map_k : lane == 1 ? &map_v : lane == 2 ? &map_q1 : lane == 3 ? &map_q2 : &map_q4) : "memory");
  if (tid == 0) {
    abort_s = 0;
    mbar_init(smem_u32(&q_full), 1);
    mbar_init(smem_u32(&q_empty), 1);
    mbar_init(smem_u32(&all_done), 1);
    for (int s = 0; s < AHEAD; ++s) mbar_init(smem_u32(&piece_full[s]), 1), mbar_init(smem_u32(&piece_empty[s]), THREADS / 32);
    for (int s = 0; s < NK; ++s) mbar_init(smem_u32(&k_full[s]), 1), mbar_init(smem_u32(&k_empty[s]), 1);
    for (int s = 0; s < NV; ++s) mbar_init(smem_u32(&v_full[s]), 1), mbar_init(smem_u32(&v_empty[s]), 1);
    for (int t = 0; t < 2; ++t) mbar_init(smem_u32(&s_full[t]), 1), mbar_init(smem_u32(&p_full[t]), 4), mbar_init(smem_u32(&o_full[t]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  ts_pdl_launch_dependents();
  const uint32_t tmem = tmem_base_s, sm = smem_u32(smem);
  volatile int* abort_flag = &abort_s;
  // The next piece of work, read where it stands; a warp gives the place back when it is done with it.  false: a wait gave up.
  int pieces = 0;
  auto fetch = [&]() -> bool { return mbar_wait(smem_u32(&piece_full[pieces % AHEAD]), (uint32_t)(pieces / AHEAD) & 1, abort_flag); };
  auto release = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&piece_empty[pieces % AHEAD]));
    ++pieces;
  };

  if (warp == 8 || warp >= 10) {
    // ---------------- copies ----------------
    // Asking for a box of 2 KB (half a head's rows of a page of 16) takes a warp 75 cycles and the copy engine under 50: three warps share every block's boxes.
    const int copier = warp == 8 ? 0 : warp - 9;
    const int box_rows = min(p.page, BN), boxes = BN / box_rows * HALVES;
    const int mine = copier + 3 * lane;  // this lane's box of a block, if it has one (11 lanes a warp at most: 32 boxes)
    const bool copies = mine < boxes;
    const int c = mine / HALVES, half = mine % HALVES;
    const uint32_t in_tile = half * ATOM + c * box_rows * 128;
    int kc = 0, vc = 0, qc = 0;
    bool ok = true;
    // The last of them plans: pieces into a ring, some ahead of the one it copies for.
    Walk<WIDE> walk;
    int planned = 0;
    bool more = copier == 2;
    if (copier == 2) {
      if (lane == 0) p.plan[2 * blockIdx.x + 1] = make_int4(0, 0, 0, 0);
      walk.begin(p, RT);
    }
    auto plan = [&](int until) {
#pragma unroll 1
      while (more && planned < until) {
        Piece piece;
        more = walk.next(p, RT, piece);
        const int at = planned % AHEAD;
        if (planned >= AHEAD && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&piece_empty[at]), (uint32_t)(planned / AHEAD - 1) & 1, abort_flag))) more = false;
        else if (lane == 0) {
          piece_s[at] = piece;
          mbar_arrive(smem_u32(&piece_full[at]));
          if (piece.nb > 0 && !piece.whole && piece.first_blk == 0) {
            p.plan[2 * blockIdx.x] = make_int4(piece.q_begin, piece.r0, piece.rows, piece.hk);
            p.plan[2 * blockIdx.x + 1] = make_int4(piece.last_cta, piece.slot, 0, 0);
          }
        }
        __syncwarp();
        ++planned;
      }
    };
    // The page of this lane's box of a block, -1 where it has none: asked for two blocks ahead, looked at when its turn comes.
    auto page_of = [&](const Piece& r, const int* table, int kb) -> int {
      const int key = kb * BN + c * box_rows, e = key / p.page;
      int page = -1;
      if (copies && key < r.n && e < p.max_blocks) page = __ldg(table + e);
      return page;
    };
    // beyond the end: the copy engine fills zeros
    auto slot_of = [&](int page, int kb) -> int {
      return page < 0 ? p.total_slots : (int)min((long long)page * p.page + (kb * BN + c * box_rows) % p.page, (long long)p.total_slots);
    };
    auto load = [&](bool keys, int slot, int hk) {
      int& count = keys ? kc : vc;
      const int stages = keys ? NK : NV, st = count % stages, use = count / stages;
      const uint32_t full = smem_u32(keys ? &k_full[st] : &v_full[st]), empty = smem_u32(keys ? &k_empty[st] : &v_empty[st]);
      if (use > 0) ok = __all_sync(0xffffffffu, mbar_wait(empty, (uint32_t)(use - 1) & 1, abort_flag));
      if (!ok) return;
      if (copier == 0 && lane == 0) mbar_expect_tx(full, TILE);  // (bytes that land before count too: the phase waits for this arrival)
      __syncwarp();
      if (copies) tma_load_3d(sm + (keys ? L::K : L::V) + st * TILE + in_tile, keys ? &map_k : &map_v, full, half * 64, hk, slot);
      ++count;
    };
    plan(1);
    while (ok) {
      ok = __all_sync(0xffffffffu, fetch());
      const Piece r = piece_s[pieces % AHEAD];
      release();
      if (!ok || r.nb == 0) break;
      const int* table = p.table + (size_t)r.b * p.max_blocks;
      int page = page_of(r, table, r.kb), ahead = r.nb > 1 ? page_of(r, table, r.kb + 1) : -1, behind = 0;
      if (copier == 1) {
        if (qc > 0) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&q_empty), (uint32_t)(qc - 1) & 1, abort_flag));
        if (ok && lane == 0) {
          // the queries: one or two tiles, or one tile's in two or four copies
          const int tiles = r.sets == 8 ? 2 : 4 / r.sets, box = r.sets >= 4 ? BM / G : r.sets == 2 ? 64 / G : 32 / G;
          mbar_expect_tx(smem_u32(&q_full), (uint32_t)(tiles * HALVES * box * G * 128));
#pragma unroll 1
          for (int i = 0; i < tiles * HALVES; ++i) {
            const int x = i / HALVES, h = i % HALVES;
            tma_load_4d(sm + L::Q + (r.sets == 8 ? x * TILE : x * r.sets * 32 * 128) + h * ATOM, r.sets >= 4 ? &map_q1 : r.sets == 2 ? &map_q2 : &map_q4, smem_u32(&q_full), h * 64,
                        0, r.hk, r.q_begin + (r.r0 + (r.sets == 8 ? x * RT : 0)) / G);
          }
        }
        __syncwarp();
        ++qc;
      }
#pragma unroll 1
      for (int s = 0; ok && s <= r.nb; ++s) {  // K of block s, V of the one before: the order in which the products need them
        const int after = s + 2 < r.nb ? page_of(r, table, r.kb + s + 2) : -1, slot = slot_of(page, r.kb + s);
        if (s < r.nb) load(true, slot, r.hk);
        if (ok && s > 0) load(false, behind, r.hk);
        if (s == 0) plan(pieces + AHEAD - 2);  // (places that the rows of the piece before the last have left: nobody waits for a copy that this warp has not asked for)
        behind = slot, page = ahead, ahead = after;
      }
    }
    if (*abort_flag) {
      // leave nothing in flight: wait (bounded, on a count of its own) for the copies already asked for
      int patience = 0;
      volatile int* own = &patience;
#pragma unroll 1
      for (int i = max(0, kc - NK); i < kc; ++i) mbar_wait(smem_u32(&k_full[i % NK]), (uint32_t)(i / NK) & 1, own);
#pragma unroll 1
      for (int i = max(0, vc - NV); i < vc; ++i) mbar_wait(smem_u32(&v_full[i % NV]), (uint32_t)(i / NV) & 1, own);
      if (qc > 0) mbar_wait(smem_u32(&q_full), (uint32_t)(qc - 1) & 1, own);
    }
  } else if (warp == 9) {
    // ---------------- products: the warp runs together, one elected lane issues ----------------
    // Items of a piece: tile i & 1, block i >> 1 for two tiles of rows, i where one tile's blocks alternate.  S of item i + 2 goes where S and P of item i lay: the
    // tensor core runs what one thread issues in order, so P V of item i has read P before.  (Two warps, one a tile, end up in step: exponentials of both tiles at
    // once and then products of both: 4 trees of 61 at 30,000 rows 330 us instead of the turns that one warp takes.)
    int ks = 0, vs = 0, qc = 0;      // stages of K and V that come next
    uint32_t kp = 0, vp = 0, pp = 0;   // and the phases that are waited for (of weights a bit per tile)
    bool ok = true;
    const uint64_t q_desc = desc_k_major(sm + L::Q), k_desc = desc_k_major(sm + L::K), v_desc = desc_mn_major(sm + L::V);
    while (ok) {
      ok = __all_sync(0xffffffffu, fetch());
      // (a reduction's result stands in a uniform register, and what is worked out from it: the operands of the products then need not be moved there one by one)
      const bool two = WIDE && __reduce_or_sync(0xffffffffu, (unsigned)piece_s[pieces % AHEAD].sets) == 8;
      const int nb = (int)__reduce_or_sync(0xffffffffu, (unsigned)piece_s[pieces % AHEAD].nb), items = two ? 2 * nb : nb;
      release();
      if (!ok || nb == 0) break;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&q_full), (uint32_t)qc & 1, abort_flag));
#pragma unroll 1
      for (int i = 0; ok && i < items + 2; ++i) {
        const int t = i & 1;
        const bool begins = !two || t == 0, ends = !two || t == 1;  // the first and the last item that reads a block
        if (i >= 2) {  // P V of item i - 2, once its weights and V are there
          bool there = true;
          if (begins) there = mbar_wait(smem_u32(&v_full[vs]), vp, abort_flag);
          there = there && mbar_wait(smem_u32(&p_full[t]), pp >> t & 1, abort_flag);
          ok = __all_sync(0xffffffffu, there);
          if (!ok) break;
          pp ^= 1u << t;
          fence_after();
          if (elect_one()) {
            const uint32_t to = 256 + t * D, from_p = t * 128;  // (the whole tensor memory is this CTA's: it begins at 0)
            const uint64_t vd = v_desc + (uint64_t)((vs * TILE) >> 4);
            umma_tmem_a(to, from_p, vd, idesc(D, true), i >= 4);
#pragma unroll
            for (int kk = 1; kk < BN / 16; ++kk) umma_tmem_a_more(to, from_p + kk * 8, vd + ((kk * 2048) >> 4), idesc(D, true));
            if (ends) umma_commit(smem_u32(&v_empty[vs]));
            if (i >= items) umma_commit(smem_u32(&o_full[t]));
            if (items == 1) umma_commit(smem_u32(&o_full[1]));  // (a tile without items: its accumulator is not read)
          }
          __syncwarp();
          if (ends && ++vs == NV) vs = 0, vp ^= 1;
        }
        if (i < items) {  // S of item i, once its K is there
          if (begins) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&k_full[ks]), kp, abort_flag));
          if (!ok) break;
          if (elect_one()) {
            const uint32_t to = t * 128;
            const uint64_t kd = k_desc + (uint64_t)((ks * TILE) >> 4), qd = q_desc + (uint64_t)(two && t ? TILE >> 4 : 0);
            umma_first(to, qd, kd, idesc(BN, false));
#pragma unroll
            for (int x = 1; x < D / 16; ++x) {
              const uint32_t off = ((x >> 2) * ATOM + (x & 3) * 32) >> 4;
              umma_more(to, qd + off, kd + off, idesc(BN, false));
            }
            umma_commit(smem_u32(&s_full[t]));
            if (ends) umma_commit(smem_u32(&k_empty[ks]));
            if (i == items - 1) umma_commit(smem_u32(&q_empty));
          }
          __syncwarp();
          if (ends && ++ks == NK) ks = 0, kp ^= 1;
        }
      }
      ++qc;
    }
    // Everything this CTA asked of the tensor core is done when this arrives, the arrivals of the commits above included: nobody leaves before.
    if (elect_one()) umma_commit(smem_u32(&all_done));
    __syncwarp();
    int patience = 0;
    mbar_wait(smem_u32(&all_done), 0, &patience);
    if (patience != 0) *abort_flag = 1;
  } else {
    // ---------------- softmax ----------------
    // (A wait that gives up raises the flag at which all later ones return at once; these warps then run to the end of the piece, barriers included, and store nothing.)
    const int t = warp >> 2, quad = warp & 3;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem + lanes + t * 128, o_addr = tmem + lanes + 256 + t * D;
    const float scale = CAP ? 1.f : p.scale_log2;
    int sc = 0, vc = 0, done = 0;
    for (;;) {
      uint32_t there = fetch();
      const Piece& r = piece_s[pieces % AHEAD];
      asm volatile(  // (all eight warps go on, or none)
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %0, 0;\n\tbarrier.cta.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "+r"(there)::"memory");
      if (!there || r.nb == 0) break;
      const int sets = r.sets, nb = r.nb, first = r.n - r.t, whole_from = r.whole_from;
      const bool two = WIDE && sets == 8;
      // this thread's row of the group
      const int in_group = (warp & (sets - 1)) * 32 + lane;
      const bool mine = two ? (t == 0 ? in_group < RT : in_group - BM < RT && RT + in_group - BM < r.rows) : in_group < r.rows;
      const int row = r.r0 + (two && t == 1 ? in_group - BM + RT : in_group);
      const int token = mine ? r.q_begin + row / G : -1;
      const int pos = mine && p.window > 0 ? p.positions[token] : 0;
      const int key0 = sets >= 4 ? 0 : sets == 2 ? (quad >> 1) * 64 : quad * 32;
      float m = -INFINITY, l = 0.f;
      const int items = two ? nb : (nb + 1 - t) / 2;
#pragma unroll 1
      for (int it = 0; it < items; ++it) {
        const int blk = two ? it : 2 * it + t, kbase = (r.kb + blk) * BN;
        mbar_wait(smem_u32(&s_full[t]), (uint32_t)sc & 1, abort_flag);
        ++sc;
        __syncwarp();
        fence_after();
        const bool open = kbase >= whole_from && kbase + BN <= first;
        if (sets >= 4)
          weigh<4, CAP>(p, r, token, pos, kbase, 0, open, s_addr, o_addr, it == 0, scale, m, l);
        else if (sets == 2)
          weigh<2, CAP>(p, r, token, pos, kbase, key0, open, s_addr, o_addr, it == 0, scale, m, l);
        else
          weigh<1, CAP>(p, r, token, pos, kbase, key0, open, s_addr, o_addr, it == 0, scale, m, l);
        if (kbase + BN > r.n) {
          // rows of V that no request has written: zeros (a masked key's weight is zero, but zero times garbage must stay zero)
          const int st = (vc + blk) % NV, bad = max(r.n - kbase, 0);
          mbar_wait(smem_u32(&v_full[st]), (uint32_t)((vc + blk) / NV) & 1, abort_flag);
          __syncwarp();
          for (int i = quad * 32 + lane; i < (BN - bad) * (D / 8); i += 128) {
            const int vrow = bad + i / (D / 8), c = i % (D / 8);
            *reinterpret_cast<uint4*>(smem + L::V + st * TILE + (c >> 3) * ATOM + vrow * 128 + ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[t]));
      }
      vc += nb;
      // ---- the group's rows ----
      mbar_wait(smem_u32(&o_full[0]), (uint32_t)done & 1, abort_flag);
      mbar_wait(smem_u32(&o_full[1]), (uint32_t)done & 1, abort_flag);
      ++done;
      ml_s[warp][lane] = make_float2(m, l);
      __syncwarp();
      fence_after();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const bool good = *abort_flag == 0;
      unsigned char* merge = smem + L::MERGE_AT;
      if (WIDE && sets == 8)
        leave<8>(p, r, good, G, RT, ml_s, merge, tmem, warp, lane);
      else if (sets == 4)
        leave<4>(p, r, good, G, RT, ml_s, merge, tmem, warp, lane);
      else if (sets == 2)
        leave<2>(p, r, good, G, RT, ml_s, merge, tmem, warp, lane);
      else
        leave<1>(p, r, good, G, RT, ml_s, merge, tmem, warp, lane);
      release();
      fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");  // (nobody reads an accumulator when the next piece's products go there)
      fence_after();
    }
  }

  fence_before();
  __syncthreads();
  if (abort_s != 0 && tid == 0) *p.error = 1;
  if (warp == 0) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// The parts of a group that fell to several CTAs: o = sum 2^(m - M) o_part / (sum 2^(m - M) l + 2^(sink - M)), the CTAs in their order.  A CTA for 32 places of
// the group whose first part is main CTA blockIdx.x's, a lane per place, a warp per 4 columns in turn.
__global__ void __launch_bounds__(256) join_tree_parts_kernel(const Params p) {
  ts_pdl_prologue();
  constexpr int VEC = D / 32;  // pieces of 4 columns per warp
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = blockIdx.x, place = blockIdx.y * 32 + lane;
  const int4 ends = p.plan[2 * c0 + 1], group = p.plan[2 * c0];
  const int c1 = ends.x;
  if (c1 <= c0) return;  // its last group was whole, or another's
  const int G = p.nq / p.nkv, RT = BM / G * G;
  const int in_tile = place % BM, in = place / BM * RT + in_tile, row = group.y + in;
  if (in_tile >= RT || in >= group.z) return;
  const int head = group.w * G + row % G;
  float top = p.head_sinks ? p.head_sinks[head] * LOG2E : -INFINITY;
  const float sink = top;
  auto part = [&](int c) -> size_t { return ((size_t)c * 2 + (c == c0 ? ends.y : 0)) * p.part_rows; };
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) top = fmaxf(top, p.part_ml[2 * (part(c) + place)]);
  float total = sink == -INFINITY ? 0.f : fast_exp2(sink - top);
  float4 o[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) {
    const size_t x = part(c);
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * (x + place));
    const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
    total += f * ml.y;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float4 y = *reinterpret_cast<const float4*>(p.part_o + x * D + ((size_t)(warp + 8 * i) * p.part_rows + place) * 4);
      o[i].x = fmaf(f, y.x, o[i].x), o[i].y = fmaf(f, y.y, o[i].y), o[i].z = fmaf(f, y.z, o[i].z), o[i].w = fmaf(f, y.w, o[i].w);
    }
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
  __nv_bfloat16* out = p.out + ((size_t)(group.x + row / G) * p.nq + head) * D;
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    *reinterpret_cast<uint2*>(out + (warp + 8 * i) * 4) = make_uint2(pack_bf16(o[i].x * inv, o[i].y * inv), pack_bf16(o[i].z * inv, o[i].w * inv));
}

// q [T, nq, D] as a 4-d tensor {D, G, nkv, T}; boxes of {64, G, 1, tokens}: the rows of a box come out ordered (token, head of the group).
int query_map(const void* ptr, long long T, int nq, int nkv, int tokens, CUtensorMap* out) {
  TsMapKey key{ptr, T, (long long)nq * 4096 + tokens, -(long long)nkv};
  std::lock_guard<std::mutex> lock(ts_map_mutex());
  auto& map_cache = ts_map_cache();
  auto it = map_cache.find(key);
  if (it != map_cache.end()) {
    *out = it->second;
    return 0;
  }
  TsEncodeTiledFn fn = ts_encode_tiled();
  if (!fn) return TS_ERR_UNSUPPORTED_SIZE;
  const int G = nq / nkv;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)G, (cuuint64_t)nkv, (cuuint64_t)T};
  cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)G * D * 2, (cuuint64_t)nq * D * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)G, 1, (cuuint32_t)tokens};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  if (fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return TS_ERR_BAD_ARGUMENT;
  if (map_cache.size() > 4096) map_cache.clear();
  map_cache.emplace(key, *out);
  return 0;
}

bool is_wide(int max_t, int nq, int nkv) { return max_t * (nq / nkv) > BM / (nq / nkv) * (nq / nkv); }

template <bool WIDE, bool CAP>
int launch(const CUtensorMap* maps, const Params& p, int max_t, cudaStream_t stream) {
  constexpr size_t smem = Layout<WIDE>::BYTES + 1024;
  const cudaError_t e = cudaFuncSetAttribute(attention_tree_kernel<WIDE, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  const int status = ts_launch(attention_tree_kernel<WIDE, CAP>, dim3(p.ctas), dim3(THREADS), smem, stream, maps[0], maps[1], maps[2], maps[3], maps[4], p);
  if (status != 0) return status;
  return ts_launch(join_tree_parts_kernel, dim3(p.ctas, p.part_rows / 32), dim3(256), 0, stream, p);
}

}  // namespace

// Whether these kernels take the sizes (those of attention_tree.cu take all).
TS_EXPORT int ts_attention_tree_tcgen05_takes(int B, int max_t, int max_context, int nq, int nkv, int page, long long num_pages, float scale) {
  if (nkv <= 0 || nq % nkv || nq / nkv > BM || B > 65535 || max_t > MAX_NODES || nkv > 65535 || !(scale > 0.f)) return 0;
  if (page < 8 || !(BN % page == 0 || page % BN == 0) || num_pages * page > 0x7fffffffLL - page) return 0;
  const long long rows = (long long)max_t * (nq / nkv), groups = rows / (BM / (nq / nkv) * (nq / nkv)) + 1;
  return (long long)B * nkv * groups * COST_TWO * ((max_context + BN - 1) / BN + 1) < (1ll << 30) ? 1 : 0;  // places of the plan fit 32 bits
}
// Floats and ints of scratch.
TS_EXPORT long long ts_attention_tree_tcgen05_scratch(int B, int max_t, int max_context, int nq, int nkv, int sms, int* ctas, int* part_rows) {
  const int G = nq / nkv, rows = max_t * G, RT = BM / G * G;
  const bool wide = is_wide(max_t, nq, nkv);
  const long long groups = (rows + (wide ? 2 * RT : RT) - 1) / (wide ? 2 * RT : RT);
  const long long blocks = (long long)B * nkv * groups * ((max_context + BN - 1) / BN);
  *ctas = (int)(blocks < 1 ? 1 : blocks < sms ? blocks : sms);
  *part_rows = wide ? 2 * BM : rows <= 32 ? 32 : rows <= 64 ? 64 : BM;
  return 2ll * *ctas * *part_rows * (D + 2) + 8ll * *ctas;
}

struct TreeArgs {
  const void *q, *k, *v;
  void* out;
  const unsigned long long* mask;
  const int *cu, *context, *table, *positions;
  const float* head_sinks;
  float* scratch;
  int* error;
  void* stream;
  long long num_pages;
  int words, max_blocks, page, T, B, max_t, nq, nkv, window, ctas, part_rows;
  float scale, cap;
};

TS_EXPORT int ts_attention_tree_tcgen05(const TreeArgs* args) {
  const auto [q, k, v, out, mask, cu, context, table, positions, head_sinks, scratch, error, stream, num_pages, words, max_blocks, page, T, B, max_t, nq, nkv, window, ctas, part_rows,
              scale, cap] = *args;
  if (B <= 0 || T <= 0) return 0;
  if (scratch == nullptr || error == nullptr || max_blocks <= 0 || ctas <= 0 || max_t <= 0 || (window > 0 && positions == nullptr)) return TS_ERR_BAD_ARGUMENT;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)scratch) % 16) return TS_ERR_BAD_ARGUMENT;
  const int G = nq / nkv;
  Params p;
  p.out = (__nv_bfloat16*)out;
  p.mask = mask, p.cu = cu, p.context = context, p.table = table, p.positions = positions, p.head_sinks = head_sinks;
  p.part_o = scratch;
  p.part_ml = scratch + 2ll * ctas * part_rows * D;
  p.plan = (int4*)(p.part_ml + 4ll * ctas * part_rows);
  p.error = error;
  p.words = words, p.max_blocks = max_blocks, p.page = page, p.nq = nq, p.nkv = nkv, p.window = window, p.num_seqs = B;
  p.total_slots = (int)(num_pages * page), p.part_rows = part_rows, p.ctas = ctas;
  p.scale_log2 = scale * LOG2E;
  p.cap_log2 = cap * LOG2E;
  p.cap_inv = cap > 0.f ? scale / cap : 0.f;
  CUtensorMap maps[5];
  const int tokens[3] = {BM / G, 64 / G > 0 ? 64 / G : 1, 32 / G > 0 ? 32 / G : 1};  // (fewer rows than a token's heads do not occur)
  for (int i = 0; i < 3; ++i) {
    const int status = query_map(q, T, nq, nkv, tokens[i], &maps[i]);
    if (status) return status;
  }
  for (int i = 0; i < 2; ++i) {
    const int status = ts_kv_cache_map(i ? v : k, num_pages * page, nkv, D, page < BN ? page : BN, &maps[3 + i]);
    if (status) return status;
  }
  const bool wide = is_wide(max_t, nq, nkv);
  cudaStream_t s = (cudaStream_t)stream;
  if (wide) return cap > 0.f ? launch<true, true>(maps, p, max_t, s) : launch<true, false>(maps, p, max_t, s);
  return cap > 0.f ? launch<false, true>(maps, p, max_t, s) : launch<false, false>(maps, p, max_t, s);
}
