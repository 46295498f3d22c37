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
// probabilities there, or, without them, 1 for x alone (then r(x) = 0 and the sum is what is left of the mass: taken off it while an eighth is left at the
// least, else added up anew over what is left, since a difference of float32 keeps no more bits than it has).  Where no child is accepted, a token is
// drawn from r by a race: the largest r_i / E_i, E_i = -ln(1 - (c_i + 1/2) / 2^24), c_i 24 bits of a hash of (key, i / 2).  With that the tokens that come out
// are distributed as if the target had been asked one by one.  Temperature 0: the argmax decides.
//
// Only the rows on the way are read: a cluster of CTAs per request, each with a piece of the vocabulary, walks down and meets once per node (maximum, sum
// and argmax of the pieces, through distributed shared memory); what is decided is decided by every CTA alike.  Sums are float32, of a few dozen
// entries a thread, joined in one order.  What bounds it is the chain of nodes: a trip to memory and a meeting each, so a thread asks for 16 entries at
// once, and the first child's row is brought to the L2 meanwhile.  The race takes its logarithm only where it may win: E >= the uniform number v that it is
// made from, so an entry with r <= best v is behind.
// Vocabulary of 151,936, float32, us on the device: one chain of 5 nodes 13.1; 32 chains of up to 6 with the drafter's probabilities 50 (59 MB, 1.2 TB/s); 16 greedy trees of 61
// nodes 27.7.
// Of that a node costs 3,500 to 7,000 cycles of scanning and 5,000 of meeting and deciding, the race 10,000 to 17,000 once (1,000 for every four entries of a thread:
// hash, exponential and comparisons; as much again where a logarithm is taken).

constexpr int QUADS = 4;                 // four entries each that a thread asks for at once
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
  int T;      // rows
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
// Four quadruples a thread at a time, VT * 4 entries from one to the next, all asked for before `use(entry, values)` works on them.  (Two CTAs of 72
// registers on an SM hide more than one of 96 that asks for the next four meanwhile.)
template <bool BF16, int VT, typename F>
__device__ __forceinline__ void scan(const void* row, int begin, int end, F use) {
  constexpr int U = QUADS, STEP = VT * 4;
  const bool vector = ((uintptr_t)row & (BF16 ? 7 : 15)) == 0;
#pragma unroll 1
  for (int at = begin; at < end; at += U * STEP) {
    float x[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) load4<BF16>(row, vector, at + u * STEP, end, x[u]);
    use(at, x);
  }
}

// e^((x - m) / T) with `rate` = log2(e) / T and x <= m, but for infinity (m is the largest number then): 1.  NaN: 0.
__device__ __forceinline__ float weight(float x, float m, float rate) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((x - m) * rate));
  return __saturatef(y);
}
// -ln(1 - (c + 1/2) / 2^24) of 24 bits c.  In float32 c + 1/2 is exact below 2^23 only; above, 2^24 - c - 1/2 = 2^e f with 1 <= f < 2 is: (24 - e) ln 2 - ln f, 17.3 for
// the largest c.  One logarithm, of 1 + z, for both (one each: a chain of five 14.9 us, of which 0.7).
__device__ __forceinline__ float waiting(uint32_t c) {
  const bool upper = c >= 1u << 23;
  const uint32_t left = __float_as_uint((float)((1u << 24) - c) - 0.5f);
  const float z = upper ? __uint_as_float((left & 0x7fffffu) | 0x3f800000u) - 1.f : ((float)c + 0.5f) * (-1.f / 16777216.f);
  return fmaf(upper ? (float)(24 + 127 - (int)(left >> 23)) : 0.f, 0.6931471805599453f, -log1pf(z));
}
// what is left of an entry with probability p and guess q after `n` refusals with the sums `total`
__device__ __forceinline__ float left_of(float p, float q, const float* total, int n) {
#pragma unroll 1
  for (int j = 0; j < n; ++j)
    if (total[j] > 0.f) p = __fdividef(fmaxf(p - q, 0.f), total[j]);
  return p;
}

// The lanes' (m, s, i), joined: m the largest with its lowest index, s the sum of s exp((m_lane - m) / T), or with `plain_sum` the plain sum.
__device__ __forceinline__ Stat join(Stat x, bool plain_sum, float inv_t) {
  float top;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(x.m));
  // (an index of -1 is none: the largest unsigned number)
  const unsigned i = __reduce_min_sync(0xffffffffu, x.m == top ? (unsigned)x.i : 0xffffffffu);
  const float s = plain_sum ? x.s : x.m == -INFINITY ? 0.f : x.s * __expf((x.m - top) * inv_t);
  return Stat{top, ts_warp_sum(s), (int)i, 0};
}
// The same over all threads of the cluster that scan: the warps of a CTA, then the CTAs, each of which leaves what it found with every other.  (As a function that is
// called a chain of five takes 13.5 us, in place 13.1.)
template <int VT>
__device__ __forceinline__ Stat meet_all(Stat x, bool scans, bool plain_sum, float inv_t, Stat* warps, Stat* met) {
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (scans) {
    const Stat w = join(x, plain_sum, inv_t);
    if (lane == 0) warps[warp] = w;
  }
  __syncthreads();
  if (warp == 0) {
    const Stat w = join(lane < VT / 32 ? warps[lane] : Stat{-INFINITY, 0.f, -1, 0}, plain_sum, inv_t);
    if (lane < C) *cluster.map_shared_rank(&met[(int)cluster.block_rank()], lane) = w;
  }
  cluster.sync();  // (the places of the next round are others: nobody writes what somebody still reads)
  return join(lane < C ? met[lane] : Stat{-INFINITY, 0.f, -1, 0}, plain_sum, inv_t);
}

// A request's nodes and where the walk stands among the children of one.
struct Nodes {
  int parent[VERIFY_MAX_NODES], token[VERIFY_MAX_NODES];
  float uniform[VERIFY_MAX_NODES];
  int child[VERIFY_MAX_NODES], children;                 // the children in their order,
  float x[VERIFY_MAX_NODES], q[VERIFY_MAX_NODES];        // their logits and the drafter's probabilities,
  float total[VERIFY_MAX_NODES];                         // and the sums of what was left behind each (with the drafter's probabilities)
  int asked, found;      // the child that is asked next, and the one that is accepted (-1: none)
  int last, whole;       // the last child that lost its mass (-1: none); a lone refusal left nothing
  float mass, added;     // without the drafter's probabilities: what is left, and the sum that it was taken off
};

// Asks the children from `asked` on, until one is accepted or what is left behind a refusal has to be added up.  One thread decides, alike in every CTA.
template <bool PROBS>
__device__ __forceinline__ void ask(Nodes& t, float most, float inv_s, int best, float inv_t, float rate, bool greedy) {
  const float added = t.added;
  const int children = t.children;
  int k = t.asked, found = -1;
  float mass = t.mass;
#pragma unroll 1
  for (; k < children; ++k) {
    const int i = t.child[k], x = t.token[i];
    bool yes;
    if (greedy) {
      yes = x == best;
    } else {
      const float p = most == -INFINITY ? 0.f : expf((t.x[k] - most) * inv_t) * inv_s;
      if (PROBS) {
        yes = t.uniform[i] * t.q[k] < left_of(p, t.q[k], t.total, k);
      } else {
        float r = added < 1.f ? weight(t.x[k], most, rate) * inv_s : p;  // (beside a sum as the sum has it: a child with all of it is accepted)
#pragma unroll 1
        for (int l = 0; l < k; ++l)
          if (t.token[t.child[l]] == x) r = 0.f;  // the same token twice: nothing is left of it
        yes = t.uniform[i] * mass < r;
        if (!yes && r > 0.f) {
          t.last = i;
          if (mass - r >= 0.125f * added) mass -= r;
          else if (k + 1 < children) break;  // (behind the last child only the race follows, which the mass does not matter to)
        }
      }
    }
    if (yes) {
      found = i;
      break;
    }
    if (PROBS && !greedy && children > 1) break;  // (the sum scales all entries of the race alike: a lone child's is not needed)
  }
  t.found = found, t.asked = k, t.mass = mass;
}

// VT threads scan, and a warp looks the children up.  With the drafter's probabilities and without them are builds apart: each is shorter (16 chains without 35.1 us in a build for
// both, 31.2), and in a build for both nvcc 12.9 took the one condition on them for true here and for false there (not with -Xcicc -O1).
template <bool BF16, bool PROBS, int VT>
__global__ void __launch_bounds__(VT + 32, VT > 512 ? 1 : 2) verify_kernel(const VerifyArgs a) {
  constexpr int VERIFY_THREADS = VT + 32;
  ts_pdl_prologue();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool scans = warp < VT / 32;
  extern __shared__ uint32_t refused_s[];  // a bit per entry of this CTA's piece: tokens that were refused at the node
  __shared__ Stat warps_s[VT / 32], met[2][MAX_CLUSTER];  // what the warps and the CTAs of the cluster found
  __shared__ Nodes tree;

  const int first = a.cu[b], nodes = first < 0 ? 0 : min(min(a.cu[b + 1], a.T) - first, min(VERIFY_MAX_NODES, a.columns));
  if (rank == 0) {
#pragma unroll 1
    for (int k = tid; k < a.columns; k += VERIFY_THREADS) a.path[(size_t)b * a.columns + k] = k == 0 && nodes > 0 ? 0 : -1, a.fresh[(size_t)b * a.columns + k] = -1;
  }
  if (nodes <= 0) {  // (all CTAs of the cluster alike)
    if (rank == 0 && tid == 0) a.counts[b] = 0;
    return;
  }
  const float T = a.temperatures[b];
  const bool greedy = !(T > 1e-10f);
  // (a row's weights are worked out on their own, everything else about T from inv_t)
  const float inv_t = greedy ? 1.f : fmaxf(1.f / T, FLT_MIN);  // (not 0: an entry of -inf has no probability at any temperature)
#pragma unroll 1
  for (int i = tid; i < nodes; i += VERIFY_THREADS) tree.parent[i] = a.parents[first + i], tree.token[i] = a.tokens[first + i], tree.uniform[i] = a.uniforms[first + i];
  const float rate = inv_t * 1.4426950408889634f;
  const int lo = rank * a.piece, hi = min(a.V, lo + a.piece), begin = lo + tid * 4;
  constexpr int ITEM = BF16 ? 2 : 4, STEP = VT * 4;
  int round = 0;
  cluster.sync();  // every CTA of the cluster has begun: its places may be written to

  auto meet = [&](float m, float s, int i, bool plain_sum) -> Stat { return meet_all<VT>(Stat{m, s, i, 0}, scans, plain_sum, inv_t, warps_s, met[round++ & 1]); };

  int here = 0, accepted = 0, token = 0;
  for (;;) {
    const unsigned char* row = reinterpret_cast<const unsigned char*>(a.logits) + (size_t)(first + here) * a.row_stride * ITEM;
    const float* guess = PROBS ? a.probs + (size_t)(first + here) * a.probs_stride : nullptr;
    float m = -INFINITY, s = 0.f;
    int mi = -1;
#pragma unroll 1
    for (int x = tid * 128; x < (hi - lo) * ITEM; x += VERIFY_THREADS * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + (size_t)lo * ITEM + x));
    if (scans) {
      // maximum, sum and argmax of the row: a thread's own running pair
      scan<BF16, VT>(row, begin, hi, [&](int at, const float (&x)[QUADS][4]) {
        float most = -INFINITY;  // (NaN is never the larger one)
#pragma unroll
        for (int u = 0; u < QUADS; ++u) most = fmaxf(most, fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3])));
        const float top = fminf(most, FLT_MAX);
        if (mi < 0 || top > m) {
          s = m == -INFINITY ? 0.f : s * __expf((m - top) * inv_t);
          m = top;
#pragma unroll
          for (int u = QUADS - 1; u >= 0; --u)
#pragma unroll
            for (int j = 3; j >= 0; --j)
              if (x[u][j] == most && at + u * STEP + j < hi) mi = at + u * STEP + j;  // (the first of equals is looked at last)
        }
        if (m > -INFINITY) {
#pragma unroll
          for (int u = 0; u < QUADS; ++u) s += (weight(x[u][0], m, rate) + weight(x[u][1], m, rate)) + (weight(x[u][2], m, rate) + weight(x[u][3], m, rate));
        }
      });
    } else {
      // the children, in their order, and their logits
      int n = 0, oldest = -1;
#pragma unroll 1
      for (int i0 = here + 1; i0 < nodes; i0 += 32) {
        const int i = i0 + lane;
        const bool mine = i < nodes && tree.parent[i] == here && tree.token[i] >= 0 && tree.token[i] < a.V;
        const unsigned all = __ballot_sync(0xffffffffu, mine);
        if (oldest < 0 && all != 0) oldest = i0 + __ffs(all) - 1;
        if (mine) {
          const int k = n + __popc(all & ((1u << lane) - 1));
          tree.child[k] = i;
          const int x = tree.token[i];
          tree.x[k] = usable(BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[x]) : reinterpret_cast<const float*>(row)[x]);
          if (PROBS) tree.q[k] = guess[x];
        }
        n += __popc(all);
      }
      if (lane == 0) tree.children = n;
      if (oldest >= 0) {  // the likeliest next row, this CTA's piece of it
        const unsigned char* ahead = reinterpret_cast<const unsigned char*>(a.logits) + ((size_t)(first + oldest) * a.row_stride + lo) * ITEM;
#pragma unroll 1
        for (int x = lane * 128; x < (hi - lo) * ITEM; x += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(ahead + x));
      }
    }
    Stat all = meet(m, s, mi, false);
    if (all.m == -INFINITY) all.i = 0;  // (nothing but NaN and -inf)
    const float inv_s = all.s > 0.f ? 1.f / all.s : 0.f;
    const int children = tree.children;  // (written before the barriers of `meet`)
    // Which child, decided alike in every CTA; with the drafter's probabilities a refusal needs the sum of what is left, without them where little is.
    if (tid == 0) tree.asked = 0, tree.whole = 0, tree.mass = tree.added = 1.f, tree.last = -1;
    float best = -1.f, bound = -1.f;  // this thread's best of the race, and the warp's
    int best_i = -1, next = -1;
    for (;;) {
      if (tid == 0) ask<PROBS>(tree, all.m, inv_s, all.i, inv_t, rate, greedy);  // (all have passed a meeting since they read what this writes)
      __syncthreads();
      next = tree.found;
      if (next >= 0 || greedy) break;
      // What follows: 0 the sum of what is left, 1 the race over it; 2: over r = max(p - q, 0) of one refused child, whose sum does not matter.
      const int asked = tree.asked, last = tree.last;
      const bool whole = tree.whole != 0;
      const int pass = asked < children ? 0 : PROBS && children == 1 && !whole ? 2 : 1;
      const bool race = pass != 0, mask = !PROBS && children > 0;
      if (mask) {
#pragma unroll 1
        for (int i = tid; i < a.piece / 32; i += VERIFY_THREADS) refused_s[i] = 0;
        __syncthreads();
#pragma unroll 1
        for (int k = tid; k < (race ? children : asked + 1); k += VERIFY_THREADS) {
          const int x = tree.token[tree.child[k]] - lo;
          if (x >= 0 && x < a.piece) atomicOr(&refused_s[x >> 5], 1u << (x & 31));
        }
        __syncthreads();
      }
      best = bound = -1.f, best_i = -1;
      float sum = 0.f;
      if (scans) {
        // Four entries a time, the next ones on their way; whole warps walk, those whose entries are behind the end too.
        const uint64_t key = a.keys[b];
        const int refusals = PROBS && !whole ? asked : 0;
        const bool row_vector = ((uintptr_t)row & (BF16 ? 7 : 15)) == 0, guess_vector = PROBS && ((uintptr_t)guess & 15) == 0;
        float x[2][4], q[2][4] = {};  // (without the drafter's probabilities zeros throughout)
        auto load = [&](int at, float (&x)[4], float (&q)[4]) {
          load4<BF16>(row, row_vector, at, hi, x);
          if (!PROBS) return;
          if (guess_vector && at + 4 <= hi) {
            const float4 w = __ldg(reinterpret_cast<const float4*>(guess + at));
            q[0] = w.x, q[1] = w.y, q[2] = w.z, q[3] = w.w;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = at + j < hi ? guess[at + j] : 0.f;
          }
        };
        load(begin, x[0], q[0]);
#pragma unroll 1
        for (int at = begin; at - lane * 4 < hi; at += STEP) {
          load(at + STEP, x[1], q[1]);
          const uint32_t out = mask && at < hi ? refused_s[(at - lo) >> 5] >> ((at - lo) & 31) : 0u;
          float r[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            r[j] = all.m == -INFINITY || ((out >> j) & 1) ? 0.f : weight(x[0][j], all.m, rate) * inv_s;
            if (pass == 2) r[j] = fmaxf(r[j] - q[0][j], 0.f);
            else if (refusals > 0) r[j] = left_of(r[j], q[0][j], tree.total, refusals);
            sum += fmaxf(r[j] - q[0][j], 0.f);
            x[0][j] = x[1][j], q[0][j] = q[1][j];
          }
          if (!race) continue;
          uint32_t c[4];
          bool may_win[4], any = false;
          const uint64_t z0 = pair_hash(key, (uint32_t)at >> 1), z1 = pair_hash(key, ((uint32_t)at >> 1) + 1);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            c[j] = (uint32_t)((j < 2 ? z0 : z1) >> (j & 1 ? 16 : 40)) & 0xFFFFFFu;
            // (from below by the upper 23 of its bits, as those of a number in [1, 2): a conversion takes longer)
            may_win[j] = at + j < hi && (best_i < 0 || r[j] > fmaf(bound, __uint_as_float(0x3f800000u | (c[j] >> 1)), -bound) * 0.999999f);
            any |= may_win[j];
          }
          if (__any_sync(0xffffffffu, any)) {
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
              const float rj = j < 2 ? (j ? r[1] : r[0]) : j == 2 ? r[2] : r[3];
              const uint32_t cj = j < 2 ? (j ? c[1] : c[0]) : j == 2 ? c[2] : c[3];
              if (j < 2 ? (j ? may_win[1] : may_win[0]) : j == 2 ? may_win[2] : may_win[3]) take_better(best, best_i, __fdividef(rj, waiting(cj)), at + j);
            }
            bound = fmaxf(bound, __uint_as_float(__reduce_max_sync(0xffffffffu, best < 0.f ? 0u : __float_as_uint(best))));
          }
        }
      }
      const Stat found = meet(best, race ? 0.f : sum, best_i, true);
      if (race) {
        token = mask && last >= 0 && !(found.m > 0.f) ? tree.token[last] : found.i;  // (nothing is left: what was refused last had it all)
        if (pass == 1 || found.m > 0.f) break;
        if (tid == 0) tree.whole = 1;  // nothing was left behind the lone refusal: as if nothing had been refused
      } else {
        if (tid == 0) tree.total[asked] = tree.mass = tree.added = found.s, tree.asked = asked + 1;
        if (mask && !(found.s > 0.f)) {
          token = tree.token[last];
          break;
        }
      }
    }
    if (next >= 0) {
      if (rank == 0 && tid == 0) {
        a.fresh[(size_t)b * a.columns + accepted] = tree.token[next];
        a.path[(size_t)b * a.columns + accepted + 1] = next;
      }
      ++accepted;
      here = next;  // (nobody but thread 0, ahead of the barrier, has read the children's places that are written again)
      continue;
    }
    if (greedy) token = max(all.i, 0);
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
// the row for all k, so it needs nobody else.  Latency bounds it: 28 layers of one request 1.9 us, 36 of 16 requests with rows of 2 KB 5.7.

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
#pragma unroll 1
  for (int k0 = 1; k0 <= count; k0 += 4) {
    long long src[4], dst[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = k0 + i, from = k <= count ? path[k] : -1;
      const bool moves = from > k && from < t;  // (else it is there already, or no node)
      src[i] = moves ? place(from) : -1;
      dst[i] = moves ? place(k) : -1;
    }
#pragma unroll 1
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
// over and over) is walked once per chain instead.  64 requests of 30,000 tokens: 8.0 us (7.7 MB, 1 TB/s: a walk of 30 places a thread and four choices of a
// chain), one of 700: 3.3.

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
#pragma unroll 1
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
#pragma unroll 1
    while (m < a.longest && m <= j && h[j - m] == suffix_s[m]) ++m;
    return m < a.shortest ? 0ull : ((unsigned long long)m << 32) | (unsigned)(j + 1);
  };
  {
    const bool vector = ((uintptr_t)h & 15) == 0;
#pragma unroll 1
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
#pragma unroll 1
  for (; chains < a.branches; ++chains) {
    unsigned long long best = 0;
    if (listed <= LISTED) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (chains > 0 && following[i] == used_s[chains - 1]) mine[i] = 0;
        best = mine[i] > best ? mine[i] : best;
      }
    } else {
#pragma unroll 1
      for (int j = tid; j < n - 1; j += LT) {
        if (h[j] != last) continue;
        const unsigned long long key = match(j);
        if (key <= best) continue;
        const int next = h[j + 1];
        bool taken = false;
#pragma unroll 1
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
#pragma unroll 1
  for (int c = 0; c < chains; ++c) {
    const int begin = begin_s[c], len = min(a.depth, n - begin);
    if (tid < len) tokens[total + tid] = h[begin + tid], parents[total + tid] = tid == 0 ? 0 : total + tid - 1;
    total += len;
  }
#pragma unroll 1
  for (int i = tid; i < width; i += LT)
    if (i == 0 || i >= total) tokens[i] = i == 0 ? last : -1, parents[i] = -1;
  if (tid == 0) a.counts[b] = total;
}

}  // namespace

TS_EXPORT int ts_verify_drafts(const VerifyArgs* args) {
  VerifyArgs a = *args;
  if (a.B <= 0) return 0;
  if (a.V <= 0 || a.columns <= 0 || a.row_stride < a.V) return TS_ERR_BAD_ARGUMENT;
  // Few requests: sixteen CTAs each, more than clusters need to run everywhere (the GPU may then be asked for it); else eight.  With an SM for every CTA (two
  // clusters of eight to each of the GPU's eight groups of SMs) as many threads as it has use for (one chain of 5: 384 threads 13.4 us, 768 13.1, 992 14.0; 16 greedy
  // trees of 61 32.2, 27.7, 30.0), else half, and two CTAs an SM (32 chains with the drafter's probabilities 49.9, with 768 threads 66).
  const int C = a.B <= 8 ? 16 : 8;
  a.piece = ((a.V + C - 1) / C + 31) / 32 * 32;
  const size_t smem = (size_t)a.piece / 8;
  if (smem > 32 * 1024 || (long long)a.B * C > (1ll << 30)) return TS_ERR_UNSUPPORTED_SIZE;
  constexpr int FEW = 768, MANY = 384;
  const bool few = (long long)a.B * C <= 128;
  const int threads = few ? FEW : MANY;
  auto kernel = a.probs != nullptr ? (few ? (a.bf16 ? verify_kernel<true, true, FEW> : verify_kernel<false, true, FEW>) : a.bf16 ? verify_kernel<true, true, MANY> : verify_kernel<false, true, MANY>)
                : few ? (a.bf16 ? verify_kernel<true, false, FEW> : verify_kernel<false, false, FEW>) : a.bf16 ? verify_kernel<true, false, MANY> : verify_kernel<false, false, MANY>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return (int)e;
  return ts_launch_cluster(kernel, dim3(a.B * C), dim3(threads + 32), smem, (cudaStream_t)a.stream, C, a);
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
