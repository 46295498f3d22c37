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
// Only the rows on the way are read: a cluster of CTAs per request, each with a piece of the vocabulary, walks down
// and meets once per node (maximum, sum and argmax of the pieces, through distributed shared memory); what is decided is decided by
// every CTA alike.  Sums are float32 over pieces of a few dozen entries a thread, joined in one order.

constexpr int VT = 512;       // threads
constexpr int MAX_CLUSTER = 16;
constexpr int VERIFY_MAX_NODES = 256;

struct VerifyArgs {
  const void* logits;
  long long row_stride;  // entries
  const float* probs;    // [T, V] with row stride probs_stride, or null
  long long probs_stride;
  const int* tokens;     // [T]
  const int* parents;    // [T], numbers inside the request
  const int* cu;         // [B + 1]
  const float* temperatures;
  const float* uniforms;  // [T]
  const unsigned long long* keys;  // [B]
  int* path;    // [B, columns]
  int* fresh;   // [B, columns]
  int* counts;  // [B]
  int V, columns, piece, bf16;  // piece: entries of the vocabulary per CTA, a multiple of 32
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
__device__ __forceinline__ float waiting_time(uint32_t bits24) { return -log1pf(-((float)bits24 + 0.5f) * (1.f / 16777216.f)); }

// Four entries from `at` on (a multiple of 4) of a row; those at or behind `end` are -inf.
__device__ __forceinline__ void load4(const VerifyArgs& a, const unsigned char* row, bool vector, int at, int end, float (&v)[4]) {
  if (a.bf16) {
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
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = usable(v[j]);
}
__device__ __forceinline__ float load1(const VerifyArgs& a, const unsigned char* row, int at) {
  return usable(a.bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[at]) : reinterpret_cast<const float*>(row)[at]);
}

// what is left of an entry with probability p and guess q after `n` refusals with the sums `total`
__device__ __forceinline__ float left_of(float p, float q, const float* total, int n) {
  for (int j = 0; j < n; ++j)
    if (total[j] > 0.f) p = __fdividef(fmaxf(p - q, 0.f), total[j]);
  return p;
}

__global__ void __launch_bounds__(VT) verify_kernel(const VerifyArgs a) {
  ts_pdl_prologue();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  extern __shared__ uint32_t refused_s[];  // a bit per entry of this CTA's piece: tokens that were refused at the node
  __shared__ Stat met[2][MAX_CLUSTER];
  __shared__ Stat of_warp[VT / 32];
  __shared__ int parent_s[VERIFY_MAX_NODES], token_s[VERIFY_MAX_NODES];
  __shared__ float child_x[VERIFY_MAX_NODES], child_q[VERIFY_MAX_NODES], uniform_s[VERIFY_MAX_NODES];
  __shared__ float total_s[VERIFY_MAX_NODES];
  __shared__ int child_s[VERIFY_MAX_NODES], children_s, next_s, refusals_s;

  const int first = a.cu[b], nodes = min(min(a.cu[b + 1] - first, VERIFY_MAX_NODES), a.columns);
  if (rank == 0) {
    for (int k = tid; k < a.columns; k += VT) a.path[(size_t)b * a.columns + k] = k == 0 && nodes > 0 ? 0 : -1, a.fresh[(size_t)b * a.columns + k] = -1;
  }
  if (nodes <= 0) {  // (all CTAs of the cluster alike)
    if (rank == 0 && tid == 0) a.counts[b] = 0;
    return;
  }
  const float T = a.temperatures[b];
  const bool greedy = !(T > 1e-10f);
  const float inv_t = greedy ? 1.f : 1.f / T;
  for (int i = tid; i < nodes; i += VT) parent_s[i] = a.parents[first + i], token_s[i] = a.tokens[first + i], uniform_s[i] = a.uniforms[first + i];
  const int lo = rank * a.piece, hi = min(a.V, lo + a.piece);
  const int item = a.bf16 ? 2 : 4;
  int round = 0;
  cluster.sync();  // every CTA of the cluster has begun: its places may be written to

  // Every CTA's (m, s, i), joined: m the largest with its lowest index, s the sum of s exp((m_piece - m) / T), or with `plain_sum` the plain sum.
  auto meet = [&](float m, float s, int i, bool plain_sum) -> Stat {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      const int i2 = __shfl_xor_sync(0xffffffffu, i, o);
      const float top = fmaxf(m, m2);
      s = plain_sum ? s + s2 : top == -INFINITY ? 0.f : s * __expf((m - top) * inv_t) + s2 * __expf((m2 - top) * inv_t);
      take_better(m, i, m2, i2);
    }
    if (lane == 0) of_warp[warp] = Stat{m, s, i, 0};
    __syncthreads();
    if (warp == 0) {
      Stat w = lane < VT / 32 ? of_warp[lane] : Stat{-INFINITY, 0.f, -1, 0};
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, w.m, o), s2 = __shfl_xor_sync(0xffffffffu, w.s, o);
        const int i2 = __shfl_xor_sync(0xffffffffu, w.i, o);
        const float top = fmaxf(w.m, m2);
        w.s = plain_sum ? w.s + s2 : top == -INFINITY ? 0.f : w.s * __expf((w.m - top) * inv_t) + s2 * __expf((m2 - top) * inv_t);
        take_better(w.m, w.i, m2, i2);
      }
      w = Stat{__shfl_sync(0xffffffffu, w.m, 0), __shfl_sync(0xffffffffu, w.s, 0), __shfl_sync(0xffffffffu, w.i, 0), 0};
      if (lane < C) *cluster.map_shared_rank(&met[round & 1][rank], lane) = w;
    }
    cluster.sync();  // (the places of the next round are others: nobody writes what somebody still reads)
    Stat out = met[round & 1][0];
    for (int c = 1; c < C; ++c) {
      const Stat w = met[round & 1][c];
      const float top = fmaxf(out.m, w.m);
      out.s = plain_sum ? out.s + w.s : top == -INFINITY ? 0.f : out.s * __expf((out.m - top) * inv_t) + w.s * __expf((w.m - top) * inv_t);
      take_better(out.m, out.i, w.m, w.i);
    }
    ++round;
    return out;
  };

  int here = 0, accepted = 0, token = 0;
  for (;;) {
    const unsigned char* row = reinterpret_cast<const unsigned char*>(a.logits) + (size_t)(first + here) * a.row_stride * item;
    const float* guess = a.probs ? a.probs + (size_t)(first + here) * a.probs_stride : nullptr;
    const bool vector = (((uintptr_t)row) & (a.bf16 ? 7 : 15)) == 0;
    if (warp == VT / 32 - 1) {  // the children, in their order, and their logits
      int n = 0;
      for (int i0 = here + 1; i0 < nodes; i0 += 32) {
        const int i = i0 + lane;
        const bool mine = i < nodes && parent_s[i] == here && token_s[i] >= 0 && token_s[i] < a.V;
        const unsigned all = __ballot_sync(0xffffffffu, mine);
        if (mine) {
          const int k = n + __popc(all & ((1u << lane) - 1));
          child_s[k] = i;
          child_x[k] = load1(a, row, token_s[i]);
          child_q[k] = guess ? guess[token_s[i]] : 1.f;
        }
        n += __popc(all);
      }
      if (lane == 0) children_s = n;
    }
    // maximum, sum and argmax of the row: a thread's own running pair
    float m = -INFINITY, s = 0.f;
    int mi = -1;
    for (int at = lo + tid * 4; at < hi; at += VT * 4) {
      float v[4];
      load4(a, row, vector, at, hi, v);
      const float top = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
      if (mi < 0 || top > m) {
        const float up = top;
        s = m == -INFINITY ? 0.f : s * __expf((m - up) * inv_t);
        m = up;
        mi = at + (v[0] == up ? 0 : v[1] == up ? 1 : v[2] == up ? 2 : 3);
      }
      if (m > -INFINITY) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s += __expf((v[j] - m) * inv_t);
      }
    }
    const Stat all = meet(m, s, mi, false);
    const float inv_s = all.s > 0.f ? 1.f / all.s : 0.f;
    const int children = children_s;  // (written before the barriers of `meet`)
    // Which child, decided alike in every CTA.
    int next = -1, refusals = 0;
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
        refusals_s = children;
      }
      __syncthreads();
      next = next_s;
      refusals = greedy || next >= 0 ? 0 : refusals_s;
    } else {
      // with the drafter's probabilities: a refusal needs the sum of what is left
      for (int k = 0; k < children && next < 0; ++k) {
        const float p = all.m == -INFINITY ? 0.f : expf((child_x[k] - all.m) * inv_t) * inv_s;
        const float r = left_of(p, child_q[k], total_s, k);
        if (uniform_s[child_s[k]] * child_q[k] < r) {
          next = child_s[k];
          break;
        }
        float sum = 0.f;
        for (int at = lo + tid * 4; at < hi; at += VT * 4) {
          float v[4];
          load4(a, row, vector, at, hi, v);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (at + j < hi && all.m > -INFINITY) {
              const float q = guess[at + j];
              sum += fmaxf(left_of(__expf((v[j] - all.m) * inv_t) * inv_s, q, total_s, k) - q, 0.f);
            }
          }
        }
        const float total = meet(0.f, sum, -1, true).s;
        __syncthreads();
        if (tid == 0) total_s[k] = total;
        __syncthreads();
      }
      refusals = next >= 0 ? 0 : children;
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
    const bool mask = guess == nullptr && refusals > 0;
    if (mask) {
      for (int i = tid; i < a.piece / 32; i += VT) refused_s[i] = 0;
      __syncthreads();
      for (int k = tid; k < refusals; k += VT) {
        const int x = token_s[child_s[k]] - lo;
        if (x >= 0 && x < a.piece) atomicOr(&refused_s[x >> 5], 1u << (x & 31));
      }
      __syncthreads();
    }
    const uint64_t key = a.keys[b];
    float best = -1.f;
    int best_i = -1;
    for (int at = lo + tid * 4; at < hi; at += VT * 4) {
      float v[4];
      load4(a, row, vector, at, hi, v);
      const uint32_t out = mask ? refused_s[(at - lo) >> 5] >> ((at - lo) & 31) : 0u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t z = pair_hash(key, (uint32_t)(at >> 1) + h);
#pragma unroll
        for (int j = 2 * h; j < 2 * h + 2; ++j) {
          if (at + j >= hi) continue;
          float r = all.m == -INFINITY || ((out >> j) & 1) ? 0.f : __expf((v[j] - all.m) * inv_t) * inv_s;
          if (guess != nullptr) r = left_of(r, guess[at + j], total_s, refusals);
          const float e = waiting_time((uint32_t)(z >> (j & 1 ? 16 : 40)) & 0xFFFFFFu);
          take_better(best, best_i, __fdividef(r, e), at + j);
        }
      }
    }
    token = meet(best, 0.f, best_i, true).i;
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
  long long num_pages;
  int columns, max_blocks, page, row_bytes;
};

template <typename W>
__global__ void __launch_bounds__(128) keep_rows_kernel(const KeepArgs a) {
  ts_pdl_prologue();
  const int b = blockIdx.y, count = min(a.counts[b], a.columns - 1);
  if (count <= 0) return;
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
  for (int k = 1; k <= count; ++k) {
    const int from = path[k];
    if (from <= k || from >= t) continue;  // already there (or no node)
    const long long src = place(from), dst = place(k);
    if (src < 0 || dst < 0) continue;
    for (int c = threadIdx.x * (int)sizeof(W); c < a.row_bytes; c += 128 * (int)sizeof(W))
      *reinterpret_cast<W*>(pool + dst + c) = *reinterpret_cast<const W*>(pool + src + c);
  }
}

// ---------------------------------------------------------------------------
// drafts from a request's own tokens
//
// m(j) = how many of the last tokens (at most `longest`) stand at j, j - 1, ... too.  Places with m(j) >= shortest, the longest match first, of
// equals the latest, give chains of what followed them, each with another first token.  A CTA per request walks its
// tokens once per chain (from the caches after the first time), for the largest (m, j).

struct LookupArgs {
  const int* history;  // [B, L], rows `stride` apart
  long long stride;
  const int* lengths;
  int* tokens;   // [B, 1 + depth * branches]
  int* parents;
  int* counts;
  int L, depth, branches, longest, shortest;
};

constexpr int LT = 1024, MAX_BRANCHES = 16, MAX_SUFFIX = 16;

__global__ void __launch_bounds__(LT) lookup_kernel(const LookupArgs a) {
  ts_pdl_prologue();
  __shared__ unsigned long long best_s[LT / 32];
  __shared__ int begin_s[MAX_BRANCHES], used_s[MAX_BRANCHES], found_s;
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
  __syncthreads();
  const int last = suffix_s[0];
  int chains = 0;
  for (; chains < a.branches; ++chains) {
    unsigned long long best = 0;  // m and j + 1
    for (int j = tid; j < n - 1; j += LT) {
      if (h[j] != last) continue;
      int m = 1;
      while (m < a.longest && m <= j && h[j - m] == suffix_s[m]) ++m;
      if (m < a.shortest) continue;
      const unsigned long long mine = ((unsigned long long)m << 32) | (unsigned)(j + 1);
      if (mine <= best) continue;
      const int following = h[j + 1];
      bool taken = false;
      for (int c = 0; c < chains; ++c) taken |= used_s[c] == following;
      if (!taken) best = mine;
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

TS_EXPORT int ts_verify_drafts(const void* logits, int bf16, long long row_stride, const float* probs, long long probs_stride, const int* tokens, const int* parents,
                               const int* cu, const float* temperatures, const float* uniforms, const unsigned long long* keys, int* path, int* fresh,
                               int* counts, int V, int B, int columns, void* stream) {
  if (B <= 0) return 0;
  if (V <= 0 || columns <= 0 || row_stride < V) return TS_ERR_BAD_ARGUMENT;
  const int C = 8;
  const int piece = ((V + C - 1) / C + 31) / 32 * 32;
  const size_t smem = (size_t)piece / 8;
  if (smem > 96 * 1024 || (long long)B * C > (1ll << 30)) return TS_ERR_UNSUPPORTED_SIZE;
  if (smem > 32 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(verify_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
  }
  VerifyArgs a{logits, row_stride, probs, probs_stride, tokens, parents, cu, temperatures, uniforms, keys, path, fresh, counts, V, columns, piece, bf16};
  return ts_launch_cluster(verify_kernel, dim3(B * C), dim3(VT), smem, (cudaStream_t)stream, C, a);
}

TS_EXPORT int ts_keep_drafted_rows(const unsigned long long* pools, int num_pools, int row_bytes, int align, long long num_pages, int page, const int* path,
                                   int columns, const int* counts, const int* cu, const int* context, const int* table, int max_blocks, int B, void* stream) {
  if (B <= 0 || num_pools <= 0 || columns <= 1) return 0;
  if (row_bytes <= 0 || page <= 0 || max_blocks <= 0 || row_bytes % align) return TS_ERR_BAD_ARGUMENT;
  if (B > 65535) return TS_ERR_UNSUPPORTED_SIZE;
  KeepArgs a{pools, path, counts, cu, context, table, num_pages, columns, max_blocks, page, row_bytes};
  const dim3 grid(num_pools, B), block(128);
  if (align == 16) return ts_launch(keep_rows_kernel<uint4>, grid, block, 0, (cudaStream_t)stream, a);
  if (align == 4) return ts_launch(keep_rows_kernel<uint32_t>, grid, block, 0, (cudaStream_t)stream, a);
  if (align == 2) return ts_launch(keep_rows_kernel<uint16_t>, grid, block, 0, (cudaStream_t)stream, a);
  return TS_ERR_BAD_ARGUMENT;
}

TS_EXPORT int ts_lookup_drafts(const int* history, long long stride, const int* lengths, int* tokens, int* parents, int* counts, int L, int B, int depth,
                               int branches, int longest, int shortest, void* stream) {
  if (B <= 0) return 0;
  if (L <= 0 || depth <= 0 || branches <= 0 || shortest < 1 || longest < shortest) return TS_ERR_BAD_ARGUMENT;
  if (branches > MAX_BRANCHES || longest > MAX_SUFFIX || depth > LT) return TS_ERR_UNSUPPORTED_SIZE;
  LookupArgs a{history, stride, lengths, tokens, parents, counts, L, depth, branches, longest, shortest};
  return ts_launch(lookup_kernel, dim3(B), dim3(LT), 0, (cudaStream_t)stream, a);
}
