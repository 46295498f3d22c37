// Drafted tokens: verification against the target's probabilities, the accepted rows of the caches, drafts looked up
// in a request's own tokens.
//
// A request brings a tree to a step: node 0 is its newest certain token, every other node a drafted one
// with a parent of a lower number.  Logits of row t are those behind node t.
#include <float.h>

#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

// ---------------------------------------------------------------------------
// verification
//
// p = softmax(logits / T) of the node the walk stands at.  Its children in the order of their numbers: child c with token x is accepted when
// u_c q(x) < r(x), r = p at first; a refused one takes its guess out of r: r <- max(r - q, 0) / sum.  q are the drafter's
// probabilities there, or, without them, 1 for x alone (then r(x) = 0 and the sum is what is left of the mass).  Where no child is accepted, a token is
// drawn from r by a race: the largest r_i / E_i, E_i = -ln(1 - (c_i + 1/2) / 2^24), c_i 24 bits of a hash of (key, i / 2).  With that the tokens that come out
// are distributed as if the target had been asked one by one.  Temperature 0: the argmax decides.
//
// Only the rows on the way are read: a cluster of CTAs per request, each with a piece of the vocabulary, walks down and meets once per node (maximum, sum
// and argmax of the pieces, through distributed shared memory); what is decided is decided by every CTA alike.  Sums are float32, of a few dozen
// entries a thread, joined in one order.  What bounds it is the chain of nodes: a trip to memory and a meeting each, so 16 entries a thread are
// asked for ahead, and the first child's row is brought to the L2 meanwhile.  The race takes its logarithm only where it may win: E >= the uniform number v that it is
// made from, so an entry with r <= best v is behind.

constexpr int VT = 512;              // threads that scan
constexpr int VERIFY_THREADS = VT + 32;  // and a warp that looks the children up
constexpr int MAX_CLUSTER = 16;
constexpr int VERIFY_MAX_NODES = 256;

struct VerifyArgs {
  const void* logits;
  const float* probs;    // [T, V] with row stride probs_stride, or null
  const int* tokens;     // [T]
  const int* parents;    // [T], numbers inside the request
  const int* cu;         // [B + 1]
  const float* temperatures;
  const float* uniforms;  // [T]
  const unsigned long long* keys;  // [B]
  int* path;    // [B, columns]
  int* fresh;   // [B, columns]
  int* counts;  // [B]
  void* stream;
  long long row_stride, probs_stride;  // entries
  int V, B, columns, bf16;
  int piece;  // entries of the vocabulary per CTA, a multiple of 32
};

struct Stat {
  float m, s;
  int i;
  int pad;
};

// the larger value wins, of equals the lower index; index -1: nothing yet
__device__ __forceinline__ void take_better(float& v, int& i, float v2, int i2) {
  if (i2 >= 0 && (i < 0 || v2 > v || (v2 == v && i2 < i))) v = v2, i = i2;
}
__device__ __forceinline__ float usable(float x) { return x == x ? fminf(x, FLT_MAX) : -INFINITY; }  // NaN: never; infinity: the largest number

__device__ __forceinline__ uint64_t pair_hash(uint64_t key, uint32_t pair) {
  uint64_t z = key ^ ((uint64_t)pair * 0xD1342543DE82EF95ull);
  z ^= z >> 32;
  z *= 0x94D049BB133111EBull;
  return z ^ (z >> 29);
}

// Four entries from `at` on (a multiple of 4) of a row; those at or behind `end` are -inf.
template <bool BF16>
__device__ __forceinline__ void load4(const void* row, bool vector, int at, int end, float (&v)[4]) {
  if (BF16) {
    const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(row);
    if (vector && at + 4 <= end) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(x + at));
      v[0] = __uint_as_float(w.x << 16), v[1] = __uint_as_float(w.x & 0xffff0000u);
      v[2] = __uint_as_float(w.y << 16), v[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = at + j < end ? __bfloat162float(x[at + j]) : -INFINITY;
    }
  } else {
    const float* x = reinterpret_cast<const float*>(row);
    if (vector && at + 4 <= end) {
      const float4 w = __ldg(reinterpret_cast<const float4*>(x + at));
      v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = at + j < end ? x[at + j] : -INFINITY;
    }
  }
}
// Four quadruples a thread, VT * 4 entries from one to the next, the next four on their way while `use(entry, values)` works on these.
template <bool BF16, typename F>
__device__ __forceinline__ void scan(const void* row, int begin, int end, F use) {
  constexpr int U = 4, STEP = VT * 4;
  const bool vector = ((uintptr_t)row & (BF16 ? 7 : 15)) == 0;
  float v[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) load4<BF16>(row, vector, begin + u * STEP, end, v[u]);
#pragma unroll 1
  for (int at = begin; at < end; at += U * STEP) {
    float x[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[u][j] = usable(v[u][j]);
    if (at + U * STEP < end) {
#pragma unroll
      for (int u = 0; u < U; ++u) load4<BF16>(row, vector, at + (U + u) * STEP, end, v[u]);
    }
    use(at, x);
  }
}

// what is left of an entry with probability p and guess q after `n` refusals with the sums `total`
__device__ __forceinline__ float left_of(float p, float q, const float* total, int n) {
  for (int j = 0; j < n; ++j)
    if (total[j] > 0.f) p = __fdividef(fmaxf(p - q, 0.f), total[j]);
  return p;
}

template <bool BF16>
__global__ void __launch_bounds__(VERIFY_THREADS) verify_kernel(const VerifyArgs a) {
  ts_pdl_prologue();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool scans = warp < VT / 32;
  extern __shared__ uint32_t refused_s[];  // a bit per entry of this CTA's piece: tokens that were refused at the node
  __shared__ Stat met[2][MAX_CLUSTER];
  __shared__ Stat of_warp[VT / 32];
  __shared__ int parent_s[VERIFY_MAX_NODES], token_s[VERIFY_MAX_NODES];
  __shared__ float child_x[VERIFY_MAX_NODES], child_q[VERIFY_MAX_NODES], uniform_s[VERIFY_MAX_NODES];
  __shared__ float total_s[VERIFY_MAX_NODES];
  __shared__ int child_s[VERIFY_MAX_NODES], children_s, next_s;

  const int first = a.cu[b], nodes = min(min(a.cu[b + 1] - first, VERIFY_MAX_NODES), a.columns);
  if (rank == 0) {
    for (int k = tid; k < a.columns; k += VERIFY_THREADS) a.path[(size_t)b * a.columns + k] = k == 0 && nodes > 0 ? 0 : -1, a.fresh[(size_t)b * a.columns + k] = -1;
  }
  if (nodes <= 0) {  // (all CTAs of the cluster alike)
    if (rank == 0 && tid == 0) a.counts[b] = 0;
    return;
  }
  const float T = a.temperatures[b];
  const bool greedy = !(T > 1e-10f);
  const float inv_t = greedy ? 1.f : 1.f / T;
  for (int i = tid; i < nodes; i += VERIFY_THREADS) parent_s[i] = a.parents[first + i], token_s[i] = a.tokens[first + i], uniform_s[i] = a.uniforms[first + i];
  const int lo = rank * a.piece, hi = min(a.V, lo + a.piece), begin = lo + tid * 4;
  constexpr int ITEM = BF16 ? 2 : 4, STEP = VT * 4;
  int round = 0;
  cluster.sync();  // every CTA of the cluster has begun: its places may be written to

  // Every CTA's (m, s, i), joined: m the largest with its lowest index, s the sum of s exp((m_piece - m) / T), or with `plain_sum` the plain sum.
  auto add = [&](Stat& x, const Stat& y, bool plain_sum) {
    const float top = fmaxf(x.m, y.m);
    x.s = plain_sum ? x.s + y.s : top == -INFINITY ? 0.f : x.s * __expf((x.m - top) * inv_t) + y.s * __expf((y.m - top) * inv_t);
    take_better(x.m, x.i, y.m, y.i);
  };
  auto meet = [&](float m, float s, int i, bool plain_sum) -> Stat {
    Stat w{m, s, i, 0};
    if (scans) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        add(w, Stat{__shfl_xor_sync(0xffffffffu, w.m, o), __shfl_xor_sync(0xffffffffu, w.s, o), __shfl_xor_sync(0xffffffffu, w.i, o), 0}, plain_sum);
      if (lane == 0) of_warp[warp] = w;
    }
    __syncthreads();
    if (warp == 0) {
      w = lane < VT / 32 ? of_warp[lane] : Stat{-INFINITY, 0.f, -1, 0};
#pragma unroll
      for (int o = VT / 64; o > 0; o >>= 1)
        add(w, Stat{__shfl_xor_sync(0xffffffffu, w.m, o), __shfl_xor_sync(0xffffffffu, w.s, o), __shfl_xor_sync(0xffffffffu, w.i, o), 0}, plain_sum);
      w = Stat{__shfl_sync(0xffffffffu, w.m, 0), __shfl_sync(0xffffffffu, w.s, 0), __shfl_sync(0xffffffffu, w.i, 0), 0};
      if (lane < C) *cluster.map_shared_rank(&met[round & 1][rank], lane) = w;
    }
    cluster.sync();  // (the places of the next round are others: nobody writes what somebody still reads)
    Stat out = met[round & 1][0];
    for (int c = 1; c < C; ++c) add(out, met[round & 1][c], plain_sum);
    ++round;
    return out;
  };

  int here = 0, accepted = 0, token = 0;
  for (;;) {
    const unsigned char* row = reinterpret_cast<const unsigned char*>(a.logits) + (size_t)(first + here) * a.row_stride * ITEM;
    const float* guess = a.probs ? a.probs + (size_t)(first + here) * a.probs_stride : nullptr;
    float m = -INFINITY, s = 0.f;
    int mi = -1;
    if (scans) {
      // maximum, sum and argmax of the row: a thread's own running pair
      scan<BF16>(row, begin, hi, [&](int at, const float (&x)[4][4]) {
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u) top = fmaxf(top, fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3])));
        if (mi < 0 || top > m) {
          s = m == -INFINITY ? 0.f : s * __expf((m - top) * inv_t);
          m = top;
#pragma unroll
          for (int u = 3; u >= 0; --u)
#pragma unroll
            for (int j = 3; j >= 0; --j)
              if (x[u][j] == top && at + u * STEP + j < hi) mi = at + u * STEP + j;  // (the first of equals is looked at last)
        }
        if (m > -INFINITY) {
#pragma unroll
          for (int u = 0; u < 4; ++u) s += (__expf((x[u][0] - m) * inv_t) + __expf((x[u][1] - m) * inv_t)) + (__expf((x[u][2] - m) * inv_t) + __expf((x[u][3] - m) * inv_t));
        }
      });
    } else {
      // the children, in their order, and their logits
      int n = 0, oldest = -1;
      for (int i0 = here + 1; i0 < nodes; i0 += 32) {
        const int i = i0 + lane;
        const bool mine = i < nodes && parent_s[i] == here && token_s[i] >= 0 && token_s[i] < a.V;
        const unsigned all = __ballot_sync(0xffffffffu, mine);
        if (oldest < 0 && all != 0) oldest = i0 + __ffs(all) - 1;
        if (mine) {
          const int k = n + __popc(all & ((1u << lane) - 1));
          child_s[k] = i;
          const int x = token_s[i];
          child_x[k] = usable(BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[x]) : reinterpret_cast<const float*>(row)[x]);
          child_q[k] = guess ? guess[x] : 1.f;
        }
        n += __popc(all);
      }
      if (lane == 0) children_s = n;
      if (oldest >= 0) {  // the likeliest next row, this CTA's piece of it
        const unsigned char* ahead = reinterpret_cast<const unsigned char*>(a.logits) + ((size_t)(first + oldest) * a.row_stride + lo) * ITEM;
        for (int x = lane * 128; x < (hi - lo) * ITEM; x += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(ahead + x));
      }
    }
    const Stat all = meet(m, s, mi, false);
    const float inv_s = all.s > 0.f ? 1.f / all.s : 0.f;
    const int children = children_s;  // (written before the barriers of `meet`)
    // Which child, decided alike in every CTA.
    int next = -1;
    if (greedy || guess == nullptr) {
      if (tid == 0) {
        float mass = 1.f;
        for (int k = 0; k < children && next < 0; ++k) {
          const int x = token_s[child_s[k]];
          if (greedy) {
            if (x == all.i) next = child_s[k];
            continue;
          }
          bool again = false;  // the same token twice: nothing is left of it
          for (int l = 0; l < k; ++l) again |= token_s[child_s[l]] == x;
          const float r = again || all.m == -INFINITY ? 0.f : expf((child_x[k] - all.m) * inv_t) * inv_s;
          if (uniform_s[child_s[k]] * mass < r)
            next = child_s[k];
          else if (mass - r > 0.f)
            mass -= r;
        }
        next_s = next;
      }
      __syncthreads();
      next = next_s;
    } else {
      // with the drafter's probabilities: a refusal needs the sum of what is left
      for (int k = 0; k < children && next < 0; ++k) {
        const float p = all.m == -INFINITY ? 0.f : expf((child_x[k] - all.m) * inv_t) * inv_s;
        const float r = left_of(p, child_q[k], total_s, k);
        if (uniform_s[child_s[k]] * child_q[k] < r) {
          next = child_s[k];
          break;
        }
        if (k + 1 == children && children == 1) break;  // (the sum scales all entries of the race alike: a lone child's is not needed)
        float sum = 0.f;
        if (scans && all.m > -INFINITY) {
          const bool vector = ((uintptr_t)guess & 15) == 0;
          scan<BF16>(row, begin, hi, [&](int at, const float (&x)[4][4]) {
            float q[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) load4<false>(guess, vector, at + u * STEP, hi, q[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (at + u * STEP + j < hi) sum += fmaxf(left_of(__expf((x[u][j] - all.m) * inv_t) * inv_s, q[u][j], total_s, k) - q[u][j], 0.f);
          });
        }
        const float total = meet(0.f, sum, -1, true).s;
        if (tid == 0) total_s[k] = total;
        __syncthreads();
      }
    }
    if (next >= 0) {
      if (rank == 0 && tid == 0) {
        a.fresh[(size_t)b * a.columns + accepted] = token_s[next];
        a.path[(size_t)b * a.columns + accepted + 1] = next;
      }
      ++accepted;
      here = next;
      __syncthreads();  // (the children's places are written again)
      continue;
    }
    if (greedy) {
      token = max(all.i, 0);
      break;
    }
    // the race over what is left
    const bool mask = guess == nullptr && children > 0;
    if (mask) {
      for (int i = tid; i < a.piece / 32; i += VERIFY_THREADS) refused_s[i] = 0;
      __syncthreads();
      for (int k = tid; k < children; k += VERIFY_THREADS) {
        const int x = token_s[child_s[k]] - lo;
        if (x >= 0 && x < a.piece) atomicOr(&refused_s[x >> 5], 1u << (x & 31));
      }
      __syncthreads();
    }
    const uint64_t key = a.keys[b];
    float best = -1.f;
    int best_i = -1;
    auto race = [&](bool lone) {
      // lone: a refused child by itself: r = max(p - q, 0), whose sum does not matter (and where it is 0, r is p)
      const bool vector = ((uintptr_t)guess & 15) == 0;
      scan<BF16>(row, begin, hi, [&](int at, const float (&x)[4][4]) {
        float q[4][4];
        if (guess != nullptr) {
#pragma unroll
          for (int u = 0; u < 4; ++u) load4<false>(guess, vector, at + u * STEP, hi, q[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = at + u * STEP;
          if (i >= hi) continue;
          const uint32_t out = mask ? refused_s[(i - lo) >> 5] >> ((i - lo) & 31) : 0u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint64_t z = pair_hash(key, (uint32_t)(i >> 1) + h);
#pragma unroll
            for (int j = 2 * h; j < 2 * h + 2; ++j) {
              if (i + j >= hi) continue;
              float r = all.m == -INFINITY || ((out >> j) & 1) ? 0.f : __expf((x[u][j] - all.m) * inv_t) * inv_s;
              if (guess != nullptr) r = lone ? fmaxf(r - q[u][j], 0.f) : left_of(r, q[u][j], total_s, children);
              const float v = ((float)((uint32_t)(z >> (j & 1 ? 16 : 40)) & 0xFFFFFFu) + 0.5f) * (1.f / 16777216.f);
              if (best_i < 0 || r > best * v) take_better(best, best_i, __fdividef(r, -log1pf(-v)), i + j);
            }
          }
        }
      });
    };
    const bool lone = guess != nullptr && children == 1;
    if (scans) race(lone);
    Stat won = meet(best, 0.f, best_i, true);
    if (lone && !(won.m > 0.f)) {  // nothing was left: as if nothing had been refused
      if (tid == 0) total_s[0] = 0.f;
      __syncthreads();
      best = -1.f, best_i = -1;
      if (scans) race(false);
      won = meet(best, 0.f, best_i, true);
    }
    token = won.i;
    break;
  }
  if (rank == 0 && tid == 0) {
    a.fresh[(size_t)b * a.columns + accepted] = token;
    a.counts[b] = accepted;
  }
}

// ---------------------------------------------------------------------------
// the accepted nodes' rows
//
// A step has stored node i's keys and values in row first + i.  Row first + path[k] moves to row first + k, k = 1 .. count, in every pool.
// The path's numbers grow, so path[k] >= k: walking k upwards nothing is written before it has been read.  A thread owns 16 bytes (or 4, 2) of
// the row for all k, so it needs nobody else.

struct KeepArgs {
  const unsigned long long* pools;  // [num_pools] addresses of the pools
  const int* path;                  // [B, columns]
  const int* counts;
  const int* cu;
  const int* context;
  const int* table;  // [B, max_blocks]
  void* stream;
  long long num_pages;
  int num_pools, columns, max_blocks, page, row_bytes, align, B;
};

// Four rows at a time: where they lie, then their bytes, are asked for before the first is written.
template <typename W>
__global__ void __launch_bounds__(128) keep_rows_kernel(const KeepArgs a) {
  ts_pdl_prologue();
  const int b = blockIdx.y, count = min(a.counts[b], a.columns - 1);
  const int t = a.cu[b + 1] - a.cu[b], first = a.context[b] - t;
  unsigned char* pool = reinterpret_cast<unsigned char*>(a.pools[blockIdx.x]);
  const int* path = a.path + (size_t)b * a.columns;
  const int* table = a.table + (size_t)b * a.max_blocks;
  auto place = [&](int node) -> long long {  // where a node's row begins; -1: it has none
    const int row = first + node;
    if (row < 0 || row / a.page >= a.max_blocks) return -1;
    const long long page = table[row / a.page];
    return page < 0 || page >= a.num_pages ? -1 : (page * a.page + row % a.page) * a.row_bytes;
  };
  for (int k0 = 1; k0 <= count; k0 += 4) {
    long long src[4], dst[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = k0 + i, from = k <= count ? path[k] : -1;
      const bool moves = from > k && from < t;  // (else it is there already, or no node)
      src[i] = moves ? place(from) : -1;
      dst[i] = moves ? place(k) : -1;
    }
    for (int c = threadIdx.x * (int)sizeof(W); c < a.row_bytes; c += 128 * (int)sizeof(W)) {
      W w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (src[i] >= 0 && dst[i] >= 0) w[i] = *reinterpret_cast<const W*>(pool + src[i] + c);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (src[i] >= 0 && dst[i] >= 0) *reinterpret_cast<W*>(pool + dst[i] + c) = w[i];
    }
  }
}

// ---------------------------------------------------------------------------
// drafts from a request's own tokens
//
// m(j) = how many of the last tokens (at most `longest`) stand at j, j - 1, ... too.  Places with m(j) >= shortest, the longest match first, of
// equals the latest, give chains of what followed them, each with another first token.  A CTA per request walks its tokens once, 16 a thread on their way, and puts
// (m, j) of the places that match into a list in shared memory, from which the chains are chosen; a request with more places than the list holds (the same few tokens
// over and over) is walked once per chain instead.

struct LookupArgs {
  const int* history;  // [B, L], rows `stride` apart
  const int* lengths;
  int* tokens;   // [B, 1 + depth * branches]
  int* parents;
  int* counts;
  void* stream;
  long long stride;
  int L, B, depth, branches, longest, shortest;
};

constexpr int LT = 1024, MAX_BRANCHES = 16, MAX_SUFFIX = 16, LISTED = 2 * LT;

__global__ void __launch_bounds__(LT) lookup_kernel(const LookupArgs a) {
  ts_pdl_prologue();
  __shared__ unsigned long long best_s[LT / 32], list_s[LISTED];
  __shared__ int begin_s[MAX_BRANCHES], used_s[MAX_BRANCHES], found_s, listed_s;
  __shared__ int suffix_s[MAX_SUFFIX];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int* h = a.history + (size_t)b * a.stride;
  const int n = min(a.lengths[b], a.L), width = 1 + a.depth * a.branches;
  int* tokens = a.tokens + (size_t)b * width;
  int* parents = a.parents + (size_t)b * width;
  if (n <= 0) {
    for (int i = tid; i < width; i += LT) tokens[i] = parents[i] = -1;
    if (tid == 0) a.counts[b] = 0;
    return;
  }
  if (tid < a.longest) suffix_s[tid] = tid < n ? h[n - 1 - tid] : -1;
  if (tid == 0) listed_s = 0;
  const int last = h[n - 1];
  __syncthreads();
  // (m, j + 1) of a place whose token is the last one, 0 where too little matches
  auto match = [&](int j) -> unsigned long long {
    int m = 1;
    while (m < a.longest && m <= j && h[j - m] == suffix_s[m]) ++m;
    return m < a.shortest ? 0ull : ((unsigned long long)m << 32) | (unsigned)(j + 1);
  };
  {
    const bool vector = ((uintptr_t)h & 15) == 0;
    for (int at = tid * 4; at < n - 1; at += 4 * LT * 4) {
      int x[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = at + u * LT * 4;
        if (vector && j + 4 <= n - 1) {
          const int4 w = *reinterpret_cast<const int4*>(h + j);
          x[u][0] = w.x, x[u][1] = w.y, x[u][2] = w.z, x[u][3] = w.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[u][i] = j + i < n - 1 ? h[j + i] : ~last;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (x[u][i] != last) continue;
          const unsigned long long key = match(at + u * LT * 4 + i);
          if (key == 0) continue;
          const int place = atomicAdd(&listed_s, 1);  // (the order does not matter: the largest are chosen)
          if (place < LISTED) list_s[place] = key;
        }
    }
  }
  __syncthreads();
  const int listed = listed_s;
  unsigned long long mine[2] = {0, 0};
  int following[2] = {0, 0};
  if (listed <= LISTED) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (tid + i * LT < listed) mine[i] = list_s[tid + i * LT], following[i] = h[(unsigned)mine[i]];
  }
  int chains = 0;
  for (; chains < a.branches; ++chains) {
    unsigned long long best = 0;
    if (listed <= LISTED) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (chains > 0 && following[i] == used_s[chains - 1]) mine[i] = 0;
        best = mine[i] > best ? mine[i] : best;
      }
    } else {
      for (int j = tid; j < n - 1; j += LT) {
        if (h[j] != last) continue;
        const unsigned long long key = match(j);
        if (key <= best) continue;
        const int next = h[j + 1];
        bool taken = false;
        for (int c = 0; c < chains; ++c) taken |= used_s[c] == next;
        if (!taken) best = key;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    if (lane == 0) best_s[warp] = best;
    __syncthreads();
    if (warp == 0) {
      best = best_s[lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
      }
      if (lane == 0) {
        found_s = best != 0;
        if (best != 0) begin_s[chains] = (int)(unsigned)best, used_s[chains] = h[(unsigned)best];
      }
    }
    __syncthreads();
    if (!found_s) break;
  }
  __syncthreads();
  int total = 1;
  for (int c = 0; c < chains; ++c) {
    const int begin = begin_s[c], len = min(a.depth, n - begin);
    if (tid < len) tokens[total + tid] = h[begin + tid], parents[total + tid] = tid == 0 ? 0 : total + tid - 1;
    total += len;
  }
  for (int i = tid; i < width; i += LT)
    if (i == 0 || i >= total) tokens[i] = i == 0 ? last : -1, parents[i] = -1;
  if (tid == 0) a.counts[b] = total;
}

}  // namespace

TS_EXPORT int ts_verify_drafts(const VerifyArgs* args) {
  VerifyArgs a = *args;
  if (a.B <= 0) return 0;
  if (a.V <= 0 || a.columns <= 0 || a.row_stride < a.V) return TS_ERR_BAD_ARGUMENT;
  // Few requests: sixteen CTAs each, more than clusters need to run everywhere (the GPU may then be asked for it); else eight.
  const int C = a.B <= 8 ? 16 : 8;
  a.piece = ((a.V + C - 1) / C + 31) / 32 * 32;
  const size_t smem = (size_t)a.piece / 8;
  if (smem > 32 * 1024 || (long long)a.B * C > (1ll << 30)) return TS_ERR_UNSUPPORTED_SIZE;
  auto kernel = a.bf16 ? verify_kernel<true> : verify_kernel<false>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return (int)e;
  return ts_launch_cluster(kernel, dim3(a.B * C), dim3(VERIFY_THREADS), smem, (cudaStream_t)a.stream, C, a);
}

TS_EXPORT int ts_keep_drafted_rows(const KeepArgs* args) {
  const KeepArgs& a = *args;
  if (a.B <= 0 || a.num_pools <= 0 || a.columns <= 1) return 0;
  if (a.row_bytes <= 0 || a.page <= 0 || a.max_blocks <= 0 || (a.align != 16 && a.align != 4 && a.align != 2) || a.row_bytes % a.align) return TS_ERR_BAD_ARGUMENT;
  if (a.B > 65535) return TS_ERR_UNSUPPORTED_SIZE;
  auto kernel = a.align == 16 ? keep_rows_kernel<uint4> : a.align == 4 ? keep_rows_kernel<uint32_t> : keep_rows_kernel<uint16_t>;
  return ts_launch(kernel, dim3(a.num_pools, a.B), dim3(128), 0, (cudaStream_t)a.stream, a);
}

TS_EXPORT int ts_lookup_drafts(const LookupArgs* args) {
  const LookupArgs& a = *args;
  if (a.B <= 0) return 0;
  if (a.L <= 0 || a.depth <= 0 || a.branches <= 0 || a.shortest < 1 || a.longest < a.shortest) return TS_ERR_BAD_ARGUMENT;
  if (a.branches > MAX_BRANCHES || a.longest > MAX_SUFFIX || a.depth > LT) return TS_ERR_UNSUPPORTED_SIZE;
  return ts_launch(lookup_kernel, dim3(a.B), dim3(LT), 0, (cudaStream_t)a.stream, a);
}
