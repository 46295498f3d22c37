// Attention of a tree of drafted tokens over the paged cache on the 5th-generation tensor cores: bfloat16, heads of 64 and 128.
//
// What it computes stands in attention_tree.cu.  A group of up to two tiles of 128 (node, query head) rows walks the keys of its request and KV head in blocks of
// 128: S = Q K^T and O += P V by tcgen05.mma with S, P and O in tensor memory, K and V brought page by page by TMA into rings.
//
// What bounds a step is reading the cache: 64 KB a block at 44 GB/s an SM are 1.5 us, the products of one tile 0.55.  The rest follows from that:
// * Persistent CTAs, each with an even share of all (request, KV head, group, block)s, worked out on the device: lengths and trees differ, and a
//   captured step serves them all.  A group whose blocks fall to several CTAs leaves parts, joined by a second kernel in a fixed order.
// * The copying warp runs ahead over the ends of groups, so that the rings stay full while a group's results leave.
// * Groups of one tile take turns on two accumulators: tile 0 the even blocks, tile 1 the odd ones, so that one block's exponentials run beside the next one's products.
// * Few rows would leave the exponentials of a block to one warp: up to 64 rows stand in the tile twice, up to 32 four times, and every copy weighs its own
//   half or quarter of the block's keys (the others' weights are zero).  The copies' sums are added when the group is done.
//
// A row's maximum is raised only when it lags more than 2^8 behind (the weights stay far inside bfloat16's range, and the division by the sum, taken with
// the same maximum, cancels it).  Weights are rounded to bfloat16 for the product with the values, their own type; sums take them unrounded.
// Every wait is bounded: one that gives up raises the error word, and the CTA ends in order.
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
constexpr uint32_t MERGE = 8 * 32 * CH * 4;
constexpr int MAX_SEQS = 1024;
constexpr int MAX_NODES = 256;
constexpr int THREADS = 352;                     // eight warps of softmax, one that copies Q and K, one that issues products, one that copies V
constexpr uint32_t SPIN_LIMIT = 1u << 22;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LAG = 8.f;
// What a block costs, in parts of a group of one tile's: shares are even in this measure.
constexpr int COST_ONE = 2, COST_TWO = 3;

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
  int* plan;              // [B + 1] what stands before each request, [B + 1]: the share of a CTA, for the joining kernel
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
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool more) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)more) : "memory");
}
// A (P, [128 rows x 16 keys], two bfloat16 per column) from tensor memory
__device__ __forceinline__ void umma_tmem_a(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool more) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)more) : "memory");
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
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
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
};
template <bool WIDE>
__device__ __forceinline__ Request request_of(const Params& p, int b, int RT) {
  Request r;
  r.q_begin = p.cu[b];
  r.t = p.cu[b + 1] - r.q_begin;
  r.n = p.context[b];
  r.rows = r.t > 0 ? r.t * (p.nq / p.nkv) : 0;
  r.groups = (r.rows + (WIDE ? 2 * RT : RT) - 1) / (WIDE ? 2 * RT : RT);
  int lo = 0;
  if (p.window > 0 && r.t > 0) {  // the first row that any node sees
    int lowest = INT_MAX;
    for (int i = 0; i < r.t; ++i) lowest = min(lowest, p.positions[r.q_begin + i]);
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

// A piece of work: blocks blk0 .. blk1 - 1 (of all `blocks`) of a group of rows.
struct Piece {
  int b, hk, g, blk0, blk1, at;  // at: where the group begins
};

// Walks over the pieces of one CTA's share [from, to).
template <bool WIDE>
struct Walk {
  int b, hk, g, from, to, at;  // at: where group (b, hk, g) begins
  Request r;
  __device__ __forceinline__ void begin(const Params& p, const int* before, int RT, int from_, int to_) {
    from = from_, to = to_;
    int lo = 0, hi = p.num_seqs;  // the last request that begins at or before `from`
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= from) lo = mid; else hi = mid;
    }
    b = lo;
    r = request_of<WIDE>(p, b, RT);
    const int head = cost_of_head<WIDE>(r, RT);
    hk = head > 0 ? min((from - before[b]) / head, p.nkv - 1) : p.nkv - 1;
    const int group = r.blocks * (WIDE ? COST_TWO : COST_ONE);
    const int rest = from - before[b] - hk * head;
    g = group > 0 ? min(rest / group, max(r.groups - 1, 0)) : 0;
    at = before[b] + hk * head + g * group;
  }
  __device__ __forceinline__ bool next(const Params& p, int RT, Piece& out) {
    while (b < p.num_seqs && at < to) {
      bool found = false;
      if (r.groups > 0) {
        const int cost = cost_of<WIDE>(r, g, RT);
        // blocks whose beginning lies in [from, to)
        const int blk0 = from > at ? (from - at + cost - 1) / cost : 0;
        const int blk1 = min(r.blocks, (to - at + cost - 1) / cost);
        found = blk0 < blk1;
        out = Piece{b, hk, g, blk0, blk1, at};
        at += r.blocks * cost;
      }
      if (found) {
        last = r;
        step(p, RT);
        return true;
      }
      step(p, RT);
    }
    return false;
  }
  Request last;  // the request of the piece that `next` gave
  __device__ __forceinline__ void step(const Params& p, int RT) {
    if (++g < r.groups) return;
    g = 0;
    if (r.groups > 0 && ++hk < p.nkv) return;
    hk = 0;
    if (++b < p.num_seqs) r = request_of<WIDE>(p, b, RT);
  }
};

// How the rows of a piece lie in the tensor memory: `sets` sets of 32 rows in different warps (8: two tiles of rows; 4, 2, 1: one tile once, twice, four times, in
// each of the two accumulators).  Warp w holds set w % sets.
__device__ __forceinline__ int sets_of(int rows_of_group, int RT) { return rows_of_group > RT ? 8 : rows_of_group > 64 ? 4 : rows_of_group > 32 ? 2 : 1; }

// Which of the 32 keys from `base` on a node sees, as bits.
__device__ __forceinline__ uint32_t seen_bits(const Params& p, const Request& r, int token, int pos, int base) {
  const int first = r.n - r.t;
  uint32_t out = 0;
  const int ahead = first - base;  // keys of these 32 ahead of the step's rows
  if (ahead > 0) {
    out = ahead >= 32 ? 0xffffffffu : (1u << ahead) - 1;
    if (p.window > 0) {
      const long long hidden = (long long)pos - p.window + 1 - base;
      out = hidden >= 32 ? 0u : hidden > 0 ? out & ~((1u << (int)hidden) - 1) : out;
    }
  }
  if (ahead < 32 && base < r.n) {
    const unsigned long long* words = p.mask + (size_t)token * p.words;
    const int from = max(-ahead, 0);  // the first node among these keys
    const int w = from >> 6, off = from & 63;
    unsigned long long x = w < p.words ? words[w] >> off : 0ull;
    if (off > 32 && w + 1 < p.words) x |= words[w + 1] << (64 - off);
    uint32_t bits = (uint32_t)x;
    const int nodes = min(r.t - from, 32);
    bits = nodes >= 32 ? bits : nodes > 0 ? bits & ((1u << nodes) - 1) : 0u;
    if (p.window > 0) {
      for (uint32_t left = bits; left != 0; left &= left - 1) {
        const int i = __ffs(left) - 1;
        if (p.positions[r.q_begin + from + i] <= pos - p.window) bits &= ~(1u << i);
      }
    }
    out |= ahead > 0 ? bits << ahead : bits;
  }
  return out;
}

// N scores of a row from column `col` of the block on, capped, and with -inf for keys that its node does not see.
template <int N, bool CAP>
__device__ __forceinline__ void scores(const Params& p, const Request& r, int token, int pos, int kbase, int col, bool open, uint32_t s_addr, uint32_t* v) {
#pragma unroll
  for (int c = 0; c < N; c += 32) tmem_ld32(s_addr + col + c, v + c);
  tmem_ld_wait();
  if (CAP) {
    // cap * tanh(x), in units of log2: tanh(x) = 1 - 2 / (exp(2x) + 1), exact at both ends, absolute error of a few 1e-7 in between
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = __float_as_uint(p.cap_log2 * (1.f - __fdividef(2.f, __expf(2.f * p.cap_inv * __uint_as_float(v[i])) + 1.f)));
  }
  if (!open) {
#pragma unroll
    for (int c = 0; c < N; c += 32) {
      const uint32_t bits = token >= 0 ? seen_bits(p, r, token, pos, kbase + col + c) : 0u;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (!((bits >> i) & 1)) v[c + i] = 0xff800000u;  // -inf
    }
  }
}
template <int N>
__device__ __forceinline__ float largest(const uint32_t* v) {
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < N; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(v[i]));
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
// N scores to N / 2 pairs of weights (in v's first half); returns their sum.
template <int N>
__device__ __forceinline__ float weights(uint32_t* v, float scale, float off) {
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float a = fast_exp2(fmaf(__uint_as_float(v[i]), scale, -off)), b = fast_exp2(fmaf(__uint_as_float(v[i + 1]), scale, -off));
    sum[i >> 1 & 3] += a + b;
    v[i >> 1] = pack_bf16(a, b);
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// One block's weights for one warp's 32 rows: KEYS keys from column `key0` of the block on.  Scores come from `s_addr` (the tile's columns at this warp's lanes); the
// weights of all 128 keys go over them as bfloat16, zeros for keys that are other copies' part.
template <int KEYS, bool CAP>
__device__ __forceinline__ void weigh(const Params& p, const Request& r, int token, int pos, int kbase, int key0, bool open, uint32_t s_addr, uint32_t o_addr,
                                      bool first_item, float& m_run, float& l_run) {
  constexpr int HELD = KEYS < 64 ? KEYS : 64;  // (of 128 the second 64 are kept and the first read again: all would not fit the registers)
  const float scale = CAP ? 1.f : p.scale_log2;
  uint32_t v[HELD];
  float m_blk = -INFINITY;
  if (KEYS == 128) {
    scores<64, CAP>(p, r, token, pos, kbase, 0, open, s_addr, v);
    m_blk = largest<64>(v);
  }
  scores<HELD, CAP>(p, r, token, pos, kbase, KEYS == 128 ? 64 : key0, open, s_addr, v);
  m_blk = fmaxf(m_blk, largest<HELD>(v)) * scale;  // (scale > 0)
  const bool raise = m_blk - m_run > LAG;          // also where m_run is -inf and m_blk is not
  if (__any_sync(0xffffffffu, raise)) {
    const float m_new = raise ? m_blk : m_run;
    const float corr = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
    m_run = m_new;
    l_run *= corr;
    if (!first_item) {
      // (the product before this one on the accumulator is complete: the scores, asked for behind it, are)
#pragma unroll
      for (int c = 0; c < D; c += 16) {
        uint32_t o[16];
        tmem_ld16(o_addr + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
        tmem_st16(o_addr + c, o);
      }
      tmem_st_wait();
    }
  }
  const float off = m_run == -INFINITY ? 0.f : m_run;
  l_run += weights<HELD>(v, scale, off);
  if (KEYS == 128) {
    uint32_t w[64];
    scores<64, CAP>(p, r, token, pos, kbase, 0, open, s_addr, w);
    l_run += weights<64>(w, scale, off);
    tmem_st32(s_addr, w);
    tmem_st32(s_addr + 32, v);
  } else if (KEYS == 64) {
    uint32_t zero[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) zero[i] = 0u;
    tmem_st32(s_addr + key0 / 2, v);
    tmem_st32(s_addr + 32 - key0 / 2, zero);
  } else {
    uint32_t zero[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) zero[i] = 0u;
#pragma unroll
    for (int c = 0; c < 64; c += 16) {
      if (c == key0 / 2) tmem_st16(s_addr + c, v);
      else tmem_st16(s_addr + c, zero);
    }
  }
  tmem_st_wait();
}

template <bool WIDE, bool CAP>
__global__ void __launch_bounds__(THREADS, 1) attention_tree_kernel(const __grid_constant__ CUtensorMap map_q1, const __grid_constant__ CUtensorMap map_q2,
                                                                    const __grid_constant__ CUtensorMap map_q4, const __grid_constant__ CUtensorMap map_k,
                                                                    const __grid_constant__ CUtensorMap map_v, const Params p) {
  using L = Layout<WIDE>;
  constexpr int NK = L::NK, NV = L::NV;
  ts_pdl_wait();  // tensor memory is never held while waiting for another kernel
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t q_full, q_empty, k_full[NK], k_empty[NK], v_full[NV], v_empty[NV], s_full[2], p_full[2], o_full[2], all_done;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;
  __shared__ int before_s[MAX_SEQS + 1], sum_s[THREADS / 32];
  __shared__ float2 ml_s[8][32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.nq / p.nkv, RT = BM / G * G;

  if (tid == 0) {
    abort_s = 0;
    mbar_init(smem_u32(&q_full), 1);
    mbar_init(smem_u32(&q_empty), 1);
    mbar_init(smem_u32(&all_done), 1);
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
  // What stands before each request: a running sum over the batch, every CTA for itself.
  int total = 0;
  for (int b0 = 0; b0 < p.num_seqs; b0 += THREADS) {
    const int b = b0 + tid;
    int mine = 0;
    if (b < p.num_seqs) mine = cost_of_head<WIDE>(request_of<WIDE>(p, b, RT), RT) * p.nkv;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) sum_s[warp] = sum;
    __syncthreads();
    int ahead = total, all = total;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) ahead += sum_s[w];
      all += sum_s[w];
    }
    if (b < p.num_seqs) before_s[b] = ahead + sum - mine;
    total = all;
    __syncthreads();
  }
  const int share = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  if (tid == 0) before_s[p.num_seqs] = total;
  fence_before();
  __syncthreads();
  fence_after();
  ts_pdl_launch_dependents();
  if (blockIdx.x == 0) {
    for (int b = tid; b <= p.num_seqs; b += THREADS) p.plan[b] = before_s[b];
    if (tid == 0) p.plan[p.num_seqs + 1] = share;
  }
  const uint32_t tmem = tmem_base_s, sm = smem_u32(smem);
  volatile int* abort_flag = &abort_s;
  const int from = min((long long)blockIdx.x * share, (long long)total), to = min((long long)from + share, (long long)total);
  Walk<WIDE> walk;
  Piece piece;
  walk.begin(p, before_s, RT, from, to);

  if (warp == 8 || warp == 10) {
    // ---------------- copies: Q and K, and V ----------------
    const bool keys = warp == 8;
    const int box_rows = min(p.page, BN), copies = BN / box_rows;
    const int c = lane / HALVES, half = lane % HALVES;  // this lane's box of a block (at most 16 a half: pages of 8)
    const int stages = keys ? NK : NV;
    uint64_t* full = keys ? k_full : v_full;
    uint64_t* empty = keys ? k_empty : v_empty;
    const uint32_t to_smem = sm + (keys ? L::K : L::V) + half * ATOM + c * box_rows * 128;
    int count = 0, qc = 0;
    bool ok = true;
    // Where this lane's box of a block lies in the cache (asked for two blocks ahead).
    auto find = [&](const Request& r, const int* table, int kb) -> int {
      const int key = kb * BN + c * box_rows, e = key / p.page;
      int slot = p.total_slots;  // beyond the end: zeros (a page that is not held)
      if (c < copies && key < r.n && e < p.max_blocks) {
        const int page = __ldg(table + e);
        if (page >= 0) slot = (int)min((long long)page * p.page + (key - e * p.page), (long long)p.total_slots);
      }
      return slot;
    };
    while (ok && walk.next(p, RT, piece)) {
      const Request r = walk.last;
      const int* table = p.table + (size_t)piece.b * p.max_blocks;
      const int nb = piece.blk1 - piece.blk0, kb = r.kb0 + piece.blk0;
      int slot = find(r, table, kb), ahead = nb > 1 ? find(r, table, kb + 1) : 0;
      if (keys) {
        const int r0 = piece.g * (WIDE ? 2 * RT : RT), rows = min(r.rows - r0, WIDE ? 2 * RT : RT), sets = sets_of(rows, RT);
        if (qc > 0) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&q_empty), (uint32_t)(qc - 1) & 1, abort_flag));
        if (!ok) break;
        if (lane == 0) {
          // the queries: one or two tiles, or one tile's in two or four copies
          const int boxes = sets == 8 ? 2 : 4 / sets, box = sets == 8 || sets == 4 ? BM / G : sets == 2 ? 64 / G : 32 / G;
          mbar_expect_tx(smem_u32(&q_full), (uint32_t)(boxes * HALVES * box * G * 128));
          for (int i = 0; i < boxes; ++i)
            for (int h = 0; h < HALVES; ++h)
              tma_load_4d(sm + L::Q + (sets == 8 ? i * TILE : i * sets * 32 * 128) + h * ATOM, sets >= 4 ? &map_q1 : sets == 2 ? &map_q2 : &map_q4, smem_u32(&q_full), h * 64, 0,
                          piece.hk, r.q_begin + (r0 + (sets == 8 ? i * RT : 0)) / G);
        }
        ++qc;
      }
      for (int s = 0; s < nb; ++s) {
        const int after = s + 2 < nb ? find(r, table, kb + s + 2) : 0;
        const int st = count % stages, use = count / stages;
        if (use > 0) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[st]), (uint32_t)(use - 1) & 1, abort_flag));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(smem_u32(&full[st]), TILE);
        __syncwarp();
        if (c < copies) tma_load_3d(to_smem + st * TILE, keys ? &map_k : &map_v, smem_u32(&full[st]), half * 64, piece.hk, slot);
        ++count;
        slot = ahead, ahead = after;
      }
    }
    if (*abort_flag) {
      // leave nothing in flight: wait (bounded, on a count of its own) for the copies already asked for
      int patience = 0;
      volatile int* own = &patience;
      for (int i = max(0, count - stages); i < count; ++i) mbar_wait(smem_u32(&full[i % stages]), (uint32_t)(i / stages) & 1, own);
      if (qc > 0) mbar_wait(smem_u32(&q_full), (uint32_t)(qc - 1) & 1, own);
    }
  } else if (warp == 9) {
    // ---------------- products: the warp runs together, one elected lane issues ----------------
    // Items of a piece: tile i & 1, block i >> 1 for two tiles of rows, i where one tile's blocks alternate.  S of item i + 2 goes where S and P of item i lay: the
    // tensor core runs what one thread issues in order, so P V of item i has read P before.
    int kc = 0, vc = 0, qc = 0, pc[2] = {0, 0};
    bool ok = true;
    const uint64_t q_desc = desc_k_major(sm + L::Q), k_desc = desc_k_major(sm + L::K), v_desc = desc_mn_major(sm + L::V);
    while (ok && walk.next(p, RT, piece)) {
      const Request r = walk.last;
      const int rows = min(r.rows - piece.g * (WIDE ? 2 * RT : RT), WIDE ? 2 * RT : RT);
      const bool two = WIDE && rows > RT;
      const int nb = piece.blk1 - piece.blk0, items = two ? 2 * nb : nb;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&q_full), (uint32_t)qc & 1, abort_flag));
      if (!ok) break;
      auto issue_s = [&](int i) {
        const int blk = two ? i >> 1 : i, st = (kc + blk) % NK;
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&k_full[st]), (uint32_t)((kc + blk) / NK) & 1, abort_flag));
        if (!ok) return;
        fence_after();
        if (elect_one()) {
          const uint64_t kd = k_desc + (uint64_t)((st * TILE) >> 4), qd = q_desc + (uint64_t)(two && (i & 1) ? TILE >> 4 : 0);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * ATOM + (ks & 3) * 32) >> 4;
            umma(tmem + (i & 1) * 128, qd + off, kd + off, idesc(BN, false), ks > 0);
          }
          umma_commit(smem_u32(&s_full[i & 1]));
          if (!two || (i & 1)) umma_commit(smem_u32(&k_empty[st]));
          if (i == items - 1) umma_commit(smem_u32(&q_empty));
        }
        __syncwarp();
      };
      issue_s(0);
      if (ok && items > 1) issue_s(1);
      for (int i = 0; ok && i < items; ++i) {
        const int blk = two ? i >> 1 : i, st = (vc + blk) % NV, t = i & 1;
        ok = mbar_wait(smem_u32(&v_full[st]), (uint32_t)((vc + blk) / NV) & 1, abort_flag);
        if (ok) ok = mbar_wait(smem_u32(&p_full[t]), (uint32_t)pc[t] & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++pc[t];
        fence_after();
        if (elect_one()) {
          const uint64_t vd = v_desc + (uint64_t)((st * TILE) >> 4);
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            umma_tmem_a(tmem + 256 + t * D, tmem + t * 128 + kk * 8, vd + ((kk * 2048) >> 4), idesc(D, true), kk > 0 || i >= 2);
          if (!two || (i & 1)) umma_commit(smem_u32(&v_empty[st]));
          if (i >= items - 2) umma_commit(smem_u32(&o_full[t]));
          if (items == 1) umma_commit(smem_u32(&o_full[1]));  // (a tile without items: its warps do not read it)
        }
        __syncwarp();
        if (i + 2 < items) issue_s(i + 2);
      }
      kc += nb, vc += nb, ++qc;
    }
    // Everything this CTA asked of the tensor core is done when this arrives, the arrivals of the commits above included: nobody leaves before.
    if (elect_one()) umma_commit(smem_u32(&all_done));
    __syncwarp();
    int patience = 0;
    mbar_wait(smem_u32(&all_done), 0, &patience);
    if (patience != 0) *abort_flag = 1;
  } else {
    // ---------------- softmax ----------------
    // (A wait that gives up raises the flag at which all later ones return at once; these warps then run to the end of their pieces, barriers included, and store nothing.)
    const int t = warp >> 2, quad = warp & 3;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem + lanes + t * 128, o_addr = tmem + lanes + 256 + t * D;
    unsigned char* merge = smem + L::MERGE_AT;
    int sc = 0, pieces = 0, vc = 0;
    while (walk.next(p, RT, piece)) {
      const Request r = walk.last;
      const int r0 = piece.g * (WIDE ? 2 * RT : RT), rows = min(r.rows - r0, WIDE ? 2 * RT : RT), sets = sets_of(rows, RT);
      const bool two = sets == 8;
      const int nb = piece.blk1 - piece.blk0, first = r.n - r.t;
      // this thread's row of the group
      const int in_group = (warp % sets) * 32 + lane;
      const bool mine = two ? (t == 0 ? in_group < RT : in_group - BM < RT && RT + in_group - BM < rows) : in_group < rows;
      const int row = r0 + (two && t == 1 ? in_group - BM + RT : in_group);
      const int token = mine ? r.q_begin + row / G : -1;
      const int pos = mine && p.window > 0 ? p.positions[token] : 0;
      const int keys = sets >= 4 ? 128 : sets * 32, key0 = sets >= 4 ? 0 : sets == 2 ? (quad >> 1) * 64 : quad * 32;
      float m = -INFINITY, l = 0.f;
      const int items = two ? nb : (nb + 1 - t) / 2;
      for (int it = 0; it < items; ++it) {
        const int blk = two ? it : 2 * it + t, kbase = (r.kb0 + piece.blk0 + blk) * BN;
        mbar_wait(smem_u32(&s_full[t]), (uint32_t)sc & 1, abort_flag);
        ++sc;
        __syncwarp();
        fence_after();
        const bool open = p.window == 0 && kbase + BN <= first;
        if (keys == 128)
          weigh<128, CAP>(p, r, token, pos, kbase, 0, open, s_addr, o_addr, it == 0, m, l);
        else if (keys == 64)
          weigh<64, CAP>(p, r, token, pos, kbase, key0, open, s_addr, o_addr, it == 0, m, l);
        else
          weigh<32, CAP>(p, r, token, pos, kbase, key0, open, s_addr, o_addr, it == 0, m, l);
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
      // ---- the group's rows: sums over a row's copies, through shared memory, as whole lines ----
      mbar_wait(smem_u32(&o_full[t]), (uint32_t)pieces & 1, abort_flag);
      ++pieces;
      __syncwarp();
      fence_after();
      ml_s[warp][lane] = make_float2(m, l);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const bool good = *abort_flag == 0;
      const bool whole = piece.blk0 == 0 && piece.blk1 == r.blocks;
      float top = -INFINITY, sum = 0.f;
      for (int w = warp % sets; w < 8; w += sets) top = fmaxf(top, ml_s[w][lane].x);
      for (int w = warp % sets; w < 8; w += sets) {
        const float2 x = ml_s[w][lane];
        if (x.x > -INFINITY) sum += x.y * fast_exp2(x.x - top);
      }
      float f = m == -INFINITY ? 0.f : fast_exp2(m - top);
      const int slot = piece.at <= from ? 0 : 1;  // a share has two groups in part at most: its first and its last
      float* part_o = p.part_o + ((size_t)blockIdx.x * 2 + slot) * p.part_rows * D;
      if (whole) {
        if (p.head_sinks != nullptr && mine) {
          const float sink = p.head_sinks[piece.hk * G + row % G] * LOG2E, over = fmaxf(top, sink);
          const float down = top == -INFINITY ? 0.f : fast_exp2(top - over);
          sum = sum * down + (sink == -INFINITY ? 0.f : fast_exp2(sink - over));
          f *= down;
        }
        f = sum > 0.f ? f / sum : 0.f;
      } else if (warp < sets && good && in_group < p.part_rows) {
        float* ml = p.part_ml + (((size_t)blockIdx.x * 2 + slot) * p.part_rows + in_group) * 2;
        ml[0] = top, ml[1] = sum;
      }
      for (int c0 = 0; c0 < D; c0 += CH) {
        uint32_t o[CH];
        if (items > 0) {
          tmem_ld16(o_addr + c0, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < CH / 4; ++i) {
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (f > 0.f) x = make_float4(__uint_as_float(o[4 * i]) * f, __uint_as_float(o[4 * i + 1]) * f, __uint_as_float(o[4 * i + 2]) * f, __uint_as_float(o[4 * i + 3]) * f);
          *reinterpret_cast<float4*>(merge + (warp * 32 + lane) * (CH * 4) + ((i ^ (lane >> 1 & 3)) << 4)) = x;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        for (int i = warp * 32 + lane; i < sets * 32 * (CH / 4); i += 256) {
          const int at = i / (CH / 4), c = i % (CH / 4), ln = at & 31;  // row `at` of the group's lanes, 16-byte piece c
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int w = at >> 5; w < 8; w += sets) {
            const float4 y = *reinterpret_cast<const float4*>(merge + (w * 32 + ln) * (CH * 4) + ((c ^ (ln >> 1 & 3)) << 4));
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
          }
          if (!good) continue;
          if (whole) {
            const bool tile1 = two && at >= BM;
            const int in = tile1 ? at - BM : at, rr = r0 + (tile1 ? RT : 0) + in;
            if (in < RT && rr < r0 + rows) {
              uint2 y;
              y.x = pack_bf16(x.x, x.y), y.y = pack_bf16(x.z, x.w);
              *reinterpret_cast<uint2*>(p.out + ((size_t)(r.q_begin + rr / G) * p.nq + piece.hk * G + rr % G) * D + c0 + c * 4) = y;
            }
          } else if (at < p.part_rows) {
            *reinterpret_cast<float4*>(part_o + (size_t)at * D + c0 + c * 4) = x;
          }
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
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

// The parts of a group that fell to several CTAs: o = sum 2^(m - M) o_part / (sum 2^(m - M) l + 2^(sink - M)), the CTAs in their order.  A warp per row.
template <bool WIDE>
__global__ void __launch_bounds__(256) join_tree_parts_kernel(const Params p) {
  ts_pdl_prologue();
  constexpr int VEC = D / 32;
  const int lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5), hk = blockIdx.y, b = blockIdx.z;
  const int G = p.nq / p.nkv, RT = BM / G * G, RG = WIDE ? 2 * RT : RT;
  if (row >= (p.cu[b + 1] - p.cu[b]) * G) return;
  const Request r = request_of<WIDE>(p, b, RT);
  const int g = row / RG, cost = cost_of<WIDE>(r, g, RT), share = p.plan[p.num_seqs + 1];
  const int at = p.plan[b] + hk * cost_of_head<WIDE>(r, RT) + g * r.blocks * (WIDE ? COST_TWO : COST_ONE);
  const int c0 = at / share, c1 = (at + (r.blocks - 1) * cost) / share;
  if (c0 == c1) return;  // (its CTA has written it)
  const int in = row - g * RG, place = in < RT ? in : BM + in - RT;
  if (place >= p.part_rows) return;
  const int head = hk * G + row % G;
  float top = p.head_sinks ? p.head_sinks[head] * LOG2E : -INFINITY;
  const float sink = top;
  auto part = [&](int c) -> size_t {  // where CTA c left its part of the row; it has one: share >= cost, or a block of it begins there
    return ((size_t)c * 2 + (at <= c * share ? 0 : 1)) * p.part_rows + place;
  };
  auto has = [&](int c) {
    const int from = c * share;
    return (from > at ? (from - at + cost - 1) / cost : 0) < min(r.blocks, (from + share - at + cost - 1) / cost);
  };
  for (int c = c0 + lane; c <= c1; c += 32)
    if (has(c)) top = fmaxf(top, p.part_ml[2 * part(c)]);
  top = ts_warp_max(top);
  float total = sink == -INFINITY ? 0.f : fast_exp2(sink - top), o[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) o[i] = 0.f;
  for (int c = c0; c <= c1; ++c) {
    if (!has(c)) continue;
    const size_t x = part(c);
    const float m = p.part_ml[2 * x];
    if (m == -INFINITY) continue;
    const float f = fast_exp2(m - top);
    total += f * p.part_ml[2 * x + 1];
    const float* from = p.part_o + x * D + lane * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = fmaf(f, from[i], o[i]);
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
  __nv_bfloat16* out = p.out + ((size_t)(r.q_begin + row / G) * p.nq + head) * D + lane * VEC;
#pragma unroll
  for (int i = 0; i < VEC; i += 2) *reinterpret_cast<uint32_t*>(out + i) = pack_bf16(o[i] * inv, o[i + 1] * inv);
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
  return ts_launch(join_tree_parts_kernel<WIDE>, dim3((max_t * (p.nq / p.nkv) + 7) / 8, p.nkv, p.num_seqs), dim3(256), 0, stream, p);
}

}  // namespace

// Whether these kernels take the sizes (the CUDA-core kernel takes all).
TS_EXPORT int ts_attention_tree_tcgen05_takes(int B, int max_t, int max_context, int nq, int nkv, int page, long long num_pages, float scale) {
  if (nkv <= 0 || nq % nkv || nq / nkv > BM || B > MAX_SEQS || max_t > MAX_NODES || nkv > 65535 || !(scale > 0.f)) return 0;
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
  return 2ll * *ctas * *part_rows * (D + 2) + B + 2;
}

TS_EXPORT int ts_attention_tree_tcgen05(const void* q, const void* k, const void* v, void* out, const unsigned long long* mask, int words, const int* cu,
                                        const int* context, const int* table, int max_blocks, int page, long long num_pages, const int* positions,
                                        const float* head_sinks, int T, int B, int max_t, int nq, int nkv, float scale, int window, float cap, int ctas,
                                        int part_rows, float* scratch, int* error, void* stream) {
  if (B <= 0 || T <= 0) return 0;
  if (scratch == nullptr || error == nullptr || max_blocks <= 0 || ctas <= 0 || max_t <= 0 || (window > 0 && positions == nullptr)) return TS_ERR_BAD_ARGUMENT;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)scratch) % 16) return TS_ERR_BAD_ARGUMENT;
  const int G = nq / nkv;
  Params p;
  p.out = (__nv_bfloat16*)out;
  p.mask = mask, p.cu = cu, p.context = context, p.table = table, p.positions = positions, p.head_sinks = head_sinks;
  p.part_o = scratch;
  p.part_ml = scratch + 2ll * ctas * part_rows * D;
  p.plan = (int*)(p.part_ml + 4ll * ctas * part_rows);
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
