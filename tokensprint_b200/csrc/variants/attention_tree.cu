// Attention of a tree of drafted tokens over the paged cache.
//
// Compiled once per head size: -DTS_HEAD_DIM=<multiple of 8, at most 256>.
//
// A request brings t tokens to a step, the nodes of a tree, and has n rows in the cache, the last t of them its nodes'.  Node i sees every row j < n - t
// (with a window: those with j > pos_i - window) and, of the step's rows, row n - t + k where bit k of its mask is set (with a window: and pos_k > pos_i - window).
//   o_i = sum_j p_ij v_j,  p_i = softmax over the rows it sees (and its head's sink) of s_ij = scale q_i k_j, or cap tanh(scale q_i k_j / cap).
// A node that sees nothing gets zeros.  Scores, maxima, sums and outputs are float32 until the end.
//
// The (node, query head of a group) pairs of a request are the rows of a tile for each KV head, so that what is read of the cache is read once for them all;
// the keys are cut into parts, a CTA each, whose results (maximum, sum, unnormalised output) a second kernel joins, always in the same order.
#include <math.h>

#include "../common.cuh"

#ifndef TS_HEAD_DIM
#error "compile with -DTS_HEAD_DIM=<head size>"
#endif
#if (TS_HEAD_DIM % 8) != 0 || TS_HEAD_DIM > 256 || TS_HEAD_DIM < 8
#error "TS_HEAD_DIM must be a multiple of 8 between 8 and 256"
#endif

namespace {

constexpr int D = TS_HEAD_DIM;
constexpr int MAX_NODES = 256;
constexpr float LOG2E = 1.4426950408889634f;

struct Params {
  const void* q;   // [T, nq, D]
  const void* k;   // [slots, nkv, D]
  const void* v;
  void* out;       // [T, nq, D]
  const unsigned long long* mask;  // [T, words]
  const int* cu;         // [B + 1]
  const int* context;    // [B]
  const int* table;      // [B, max_blocks]
  const int* positions;  // [T], read with a window only
  const float* head_sinks;  // [nq] or null
  float* part_o;         // [T * nq, splits, D]
  float* part_ml;        // [T * nq, splits, 2]
  int words, max_blocks, page, nq, nkv, window, splits, num_seqs, tokens;
  int num_pages;
  float scale, cap;      // cap 0: none
};

// A score in units of log2: what enters 2^x.
__device__ __forceinline__ float score_log2(const Params& p, float dot) {
  if (p.cap > 0.f) return p.cap * LOG2E * tanhf(dot * (p.scale / p.cap));
  return dot * (p.scale * LOG2E);
}

// Whether the token (global number `token`, position `pos`) of a request whose nodes begin at token q_begin and at row `first` sees row j of n.
__device__ __forceinline__ bool sees(const Params& p, int token, int pos, int j, int n, int first, int q_begin) {
  if (j >= n) return false;
  const int node = j - first;
  if (node < 0) return p.window == 0 || j > pos - p.window;
  if ((node >> 6) >= p.words || !((p.mask[(size_t)token * p.words + (node >> 6)] >> (node & 63)) & 1)) return false;
  return p.window == 0 || p.positions[q_begin + node] > pos - p.window;
}

// ---------------------------------------------------------------------------
// CUDA cores, both types: 16 RPT rows against blocks of 64 keys, RPT x 4 scores and RPT x D/16 outputs a thread.  Arithmetic in float32.

constexpr int BN = 64, TH = 256;
constexpr int KS = D + 4;  // row of keys in shared memory: 16-byte pieces of 8 neighbouring rows lie in different banks
constexpr int PS = BN + 4;
constexpr int DC = (D + 63) / 64;  // 16-byte pieces of an output row per thread

template <int RPT>
constexpr int rows_smem() { return (16 * RPT * KS + BN * KS + BN * D + 16 * RPT * PS) * 4 + 2 * BN * 8; }

__device__ __forceinline__ void copy16(float* dst, const void* src, bool there) {
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
  const int bytes = there ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(bytes) : "memory");
}

// A block's rows into shared memory; `slots`: where each begins in the pool, in entries, or -1.
template <typename T>
__device__ __forceinline__ void load_rows(float* dst, int stride, const T* pool, const long long* slots) {
  if constexpr (sizeof(T) == 4) {
    for (int i = threadIdx.x; i < BN * (D / 4); i += TH) {
      const int r = i / (D / 4), c = i % (D / 4) * 4;
      const long long at = slots[r];
      copy16(dst + r * stride + c, pool + (at < 0 ? 0 : at + c), at >= 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  } else {
    for (int i = threadIdx.x; i < BN * (D / 8); i += TH) {
      const int r = i / (D / 8), c = i % (D / 8) * 8;
      const long long at = slots[r];
      const uint4 w = at < 0 ? make_uint4(0u, 0u, 0u, 0u) : *reinterpret_cast<const uint4*>(pool + at + c);
      float4* to = reinterpret_cast<float4*>(dst + r * stride + c);
      to[0] = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
      to[1] = make_float4(__uint_as_float(w.z << 16), __uint_as_float(w.z & 0xffff0000u), __uint_as_float(w.w << 16), __uint_as_float(w.w & 0xffff0000u));
    }
  }
}
template <typename T, int LEFT>
__device__ __forceinline__ void rows_landed() {
  if constexpr (sizeof(T) == 4) asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
  __syncthreads();
}

// two float32 in one 64-bit register, and their packed product and sum: twice the work of a scalar instruction, whose three operands the registers deliver 2.6
// times a cycle and SM, the packed one's 1.9 times
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ ulonglong2 load_pairs(const float* x) { return *reinterpret_cast<const ulonglong2*>(x); }

// The first row of the cache that any token of the request sees (0 without a window), worked out by one warp.
__device__ __forceinline__ int first_row(const Params& p, int q_begin, int t, int first) {
  if (p.window == 0) return 0;
  int lowest = INT_MAX;
  for (int i = threadIdx.x & 31; i < t; i += 32) lowest = min(lowest, p.positions[q_begin + i]);
  for (int o = 16; o > 0; o >>= 1) lowest = min(lowest, __shfl_xor_sync(0xffffffffu, lowest, o));
  const long long lo = (long long)lowest - p.window + 1;
  return (int)(lo < 0 ? 0 : lo > first ? max(first, 0) : lo);
}

template <typename T, int RPT>
__global__ void __launch_bounds__(TH) tree_rows_kernel(const Params p) {
  ts_pdl_prologue();
  extern __shared__ __align__(16) float smem[];
  constexpr int RM = 16 * RPT;
  float* Qs = smem;
  float* Ks = Qs + RM * KS;
  float* Vs = Ks + BN * KS;
  float* Ps = Vs + BN * D;
  long long* slots_s = reinterpret_cast<long long*>(Ps + RM * PS);  // [2][BN]
  __shared__ int lo_s;
  const int split = blockIdx.x, hk = blockIdx.y % p.nkv, tile = blockIdx.y / p.nkv, b = blockIdx.z;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int q_begin = p.cu[b], t = p.cu[b + 1] - q_begin, n = p.context[b], first = n - t;
  const int G = p.nq / p.nkv, rows = t * G, r0 = tile * RM;
  if (t <= 0 || r0 >= rows) return;
  if (tid < 32) {
    const int lo = first_row(p, q_begin, t, first);
    if (tid == 0) lo_s = lo;
  }
  // queries: row r of the tile is token r / G, head r % G
  const T* q = reinterpret_cast<const T*>(p.q);
  for (int i = tid; i < RM * D; i += TH) {
    const int r = r0 + i / D, c = i % D;
    Qs[i / D * KS + c] = r < rows ? ts_to_float(q[((size_t)(q_begin + r / G) * p.nq + hk * G + r % G) * D + c]) : 0.f;
  }
  __syncthreads();
  // this CTA's blocks of keys: an even share of the request's
  const int kb0 = lo_s / BN, blocks = n > 0 ? (n - 1) / BN - kb0 + 1 : 0;
  const int per = (blocks + p.splits - 1) / p.splits, begin = kb0 + split * per, end = min(kb0 + blocks, begin + per);
  const int* table = p.table + (size_t)b * p.max_blocks;
  auto find_slots = [&](int blk) {
    if (tid < BN) {
      const int j = blk * BN + tid, e = j / p.page;
      long long at = -1;
      if (j < n && e < p.max_blocks) {
        const int page = table[e];
        if (page >= 0 && page < p.num_pages) at = (((long long)page * p.page + j % p.page) * p.nkv + hk) * D;
      }
      slots_s[(blk & 1) * BN + tid] = at;
    }
  };
  int token[RPT], pos[RPT];
  float m[RPT], l[RPT];
  uint64_t o[RPT][DC * 2];  // pairs of columns
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = r0 + ty * RPT + i;
    token[i] = r < rows ? q_begin + r / G : -1;
    pos[i] = token[i] >= 0 && p.window > 0 ? p.positions[token[i]] : 0;
    m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DC * 2; ++c) o[i][c] = 0ull;
  }
  const T* K = reinterpret_cast<const T*>(p.k);
  const T* V = reinterpret_cast<const T*>(p.v);
  if (begin < end) {
    find_slots(begin);
    __syncthreads();
    load_rows<T>(Ks, KS, K, slots_s + (begin & 1) * BN);
    load_rows<T>(Vs, D, V, slots_s + (begin & 1) * BN);
  }
  for (int blk = begin; blk < end; ++blk) {
    const bool more = blk + 1 < end;
    if (more) find_slots(blk + 1);
    rows_landed<T, 1>();
    uint64_t sum2[RPT][4];  // of even and of odd entries
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum2[i][j] = 0ull;
#pragma unroll 4
    for (int c = 0; c < D; c += 4) {
      ulonglong2 a[RPT], k4[4];
#pragma unroll
      for (int i = 0; i < RPT; ++i) a[i] = load_pairs(Qs + (ty * RPT + i) * KS + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) k4[j] = load_pairs(Ks + (tx + 16 * j) * KS + c);
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum2[i][j] = fma2(a[i].y, k4[j].y, fma2(a[i].x, k4[j].x, sum2[i][j]));
    }
    float s[RPT][4];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = unpack2(sum2[i][j]).x + unpack2(sum2[i][j]).y;
    __syncthreads();  // the keys have been read
    if (more) load_rows<T>(Ks, KS, K, slots_s + ((blk + 1) & 1) * BN);
    // seen by every token: rows before the step, and none that a window may hide
    const bool open = blk * BN + BN <= first && p.window == 0;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = blk * BN + tx + 16 * j;
        const bool seen = token[i] >= 0 && (open || sees(p, token[i], pos[i], key, n, first, q_begin));
        s[i][j] = seen ? score_log2(p, s[i][j]) : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float m_new = fmaxf(m[i], top);
      const float corr = m_new == -INFINITY ? 1.f : exp2f(m[i] - m_new);
      m[i] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = s[i][j] == -INFINITY ? 0.f : exp2f(s[i][j] - m_new);
        Ps[(ty * RPT + i) * PS + tx + 16 * j] = w;
        sum += w;
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l[i] = l[i] * corr + sum;
#pragma unroll
      for (int c = 0; c < DC * 2; ++c) {
        const float2 x = unpack2(o[i][c]);
        o[i][c] = pack2(x.x * corr, x.y * corr);
      }
    }
    if (more)
      rows_landed<T, 1>();
    else
      rows_landed<T, 0>();
#pragma unroll 2
    for (int k = 0; k < BN; k += 4) {
      float4 w[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) w[i] = *reinterpret_cast<const float4*>(Ps + (ty * RPT + i) * PS + k);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          const int col = tx * 4 + 64 * c;
          if (D % 64 != 0 && col >= D) continue;
          const ulonglong2 v4 = load_pairs(Vs + (k + kk) * D + col);
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float x = kk == 0 ? w[i].x : kk == 1 ? w[i].y : kk == 2 ? w[i].z : w[i].w;
            const uint64_t x2 = pack2(x, x);
            o[i][2 * c] = fma2(x2, v4.x, o[i][2 * c]);
            o[i][2 * c + 1] = fma2(x2, v4.y, o[i][2 * c + 1]);
          }
        }
      }
    }
    __syncthreads();  // the values and the weights have been read
    if (more) load_rows<T>(Vs, D, V, slots_s + ((blk + 1) & 1) * BN);
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    if (token[i] < 0) continue;
    const int head = hk * G + (r0 + ty * RPT + i) % G;
    const size_t row = (size_t)token[i] * p.nq + head;
    if (p.splits > 1) {
      const size_t at = row * p.splits + split;
      if (tx == 0) p.part_ml[2 * at] = m[i], p.part_ml[2 * at + 1] = l[i];
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const int col = tx * 4 + 64 * c;
        if (D % 64 == 0 || col < D) *reinterpret_cast<ulonglong2*>(p.part_o + at * D + col) = make_ulonglong2(o[i][2 * c], o[i][2 * c + 1]);
      }
    } else {
      float total = l[i], f = 1.f;
      if (p.head_sinks != nullptr) {
        const float sink = p.head_sinks[head] * LOG2E, top = fmaxf(m[i], sink);
        f = m[i] == -INFINITY ? 0.f : exp2f(m[i] - top);
        total = total * f + (sink == -INFINITY ? 0.f : exp2f(sink - top));
      }
      const float inv = total > 0.f ? f / total : 0.f;
      T* out = reinterpret_cast<T*>(p.out) + row * D;
#pragma unroll
      for (int c = 0; c < DC * 4; ++c) {
        const int col = tx * 4 + 64 * (c / 4) + c % 4;
        if (D % 64 == 0 || col < D) out[col] = ts_from_float<T>((c % 2 ? unpack2(o[i][c / 2]).y : unpack2(o[i][c / 2]).x) * inv);
      }
    }
  }
}

// The parts of a row: o = sum_s 2^(m_s - M) o_s / (sum_s 2^(m_s - M) l_s + 2^(sink - M)).  A warp per row, always in the same order.
template <typename T>
__global__ void __launch_bounds__(128) join_parts_kernel(const Params p) {
  ts_pdl_prologue();
  const int lane = threadIdx.x & 31;
  const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int token = (int)(row / p.nq), head = (int)(row % p.nq);
  if (token >= p.tokens || token >= p.cu[p.num_seqs]) return;  // (rows behind the last request are left as they are)
  const float* ml = p.part_ml + 2 * row * p.splits;
  float top = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, ml[2 * s]);
  top = ts_warp_max(top);
  const float sink = p.head_sinks ? p.head_sinks[head] * LOG2E : -INFINITY;
  top = fmaxf(top, sink);
  float total = sink == -INFINITY ? 0.f : exp2f(sink - top);
  float o[(D + 31) / 32];
#pragma unroll
  for (int c = 0; c < (D + 31) / 32; ++c) o[c] = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float m = ml[2 * s];
    if (m == -INFINITY) continue;
    const float f = exp2f(m - top);
    total += f * ml[2 * s + 1];
#pragma unroll
    for (int c = 0; c < (D + 31) / 32; ++c)
      if (D % 32 == 0 || c * 32 + lane < D) o[c] = fmaf(f, p.part_o[(row * p.splits + s) * D + c * 32 + lane], o[c]);
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
  T* out = reinterpret_cast<T*>(p.out) + row * D;
#pragma unroll
  for (int c = 0; c < (D + 31) / 32; ++c)
    if (D % 32 == 0 || c * 32 + lane < D) out[c * 32 + lane] = ts_from_float<T>(o[c] * inv);
}

template <typename T, int RPT>
int launch_rows(const Params& p, int B, int tiles, cudaStream_t stream) {
  constexpr int smem = rows_smem<RPT>();
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(tree_rows_kernel<T, RPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
  }
  return ts_launch(tree_rows_kernel<T, RPT>, dim3(p.splits, tiles * p.nkv, B), dim3(TH), smem, stream, p);
}

template <typename T>
int run_rows(const Params& p, int B, int max_t, cudaStream_t stream) {
  const int rows = max_t * (p.nq / p.nkv);
  const int rpt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int tiles = (rows + 16 * rpt - 1) / (16 * rpt);
  if ((long long)tiles * p.nkv > 65535 || B > 65535) return TS_ERR_UNSUPPORTED_SIZE;
  int status = rpt == 1 ? launch_rows<T, 1>(p, B, tiles, stream) : rpt == 2 ? launch_rows<T, 2>(p, B, tiles, stream) : launch_rows<T, 4>(p, B, tiles, stream);
  if (status != 0 || p.splits == 1) return status;
  return ts_launch(join_parts_kernel<T>, dim3(((size_t)p.tokens * p.nq + 3) / 4), dim3(128), 0, stream, p);
}

}  // namespace

TS_EXPORT int ts_attention_tree_head_dim() { return D; }

// In how many parts the CUDA-core kernel cuts the keys of a request of `max_context` rows: the fewest blocks in a row, counting every wave of CTAs (as many as
// registers and shared memory let run at once) and one and a half blocks for a CTA's start and the joining of its part.  (4 requests of 12,000 rows, 16 nodes, float32:
// 4 parts 567 us, one wave; 5 to 6 parts 770, two; the same work in 10 parts 692.)
TS_EXPORT int ts_attention_tree_splits(int B, int max_t, int nq, int nkv, int max_context) {
  const int rows = max_t * (nq / nkv), rpt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const long long units = (long long)B * nkv * ((rows + 16 * rpt - 1) / (16 * rpt));
  const int blocks = (max_context + BN - 1) / BN;
  const int smem = rpt == 1 ? rows_smem<1>() : rpt == 2 ? rows_smem<2>() : rows_smem<4>();
  const int by_smem = 227 * 1024 / (smem + 1024), by_registers = rpt == 1 ? 4 : D > 128 ? (rpt == 2 ? 2 : 1) : rpt == 2 ? 3 : 2;
  const long long slots = 148ll * (by_smem < by_registers ? by_smem : by_registers);
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 64 && s <= (blocks < 1 ? 1 : blocks); ++s) {
    const double cost = (double)((units * s + slots - 1) / slots) * ((blocks + s - 1) / s + 1.5);
    if (s == 1 || cost < 0.98 * least) best = s, least = cost;
  }
  return best;
}

// `tokens`: rows of q.  part: floats of scratch, tokens * nq * splits * (D + 2), where splits > 1.
TS_EXPORT int ts_attention_tree(const void* q, const void* k, const void* v, void* out, int bf16, const unsigned long long* mask, int words, const int* cu,
                                const int* context, const int* table, int max_blocks, int page, int num_pages, const int* positions, const float* head_sinks,
                                int tokens, int B, int max_t, int nq, int nkv, float scale, int window, float cap, int splits, float* part, void* stream) {
  if (B <= 0 || tokens <= 0 || max_t <= 0) return 0;
  if (nkv <= 0 || nq % nkv || page <= 0 || splits < 1 || (splits > 1 && part == nullptr) || (window > 0 && positions == nullptr)) return TS_ERR_BAD_ARGUMENT;
  if (max_t > MAX_NODES || max_t > 64 * words) return TS_ERR_UNSUPPORTED_SIZE;
  Params p{q, k, v, out, mask, cu, context, table, positions, head_sinks, part, nullptr, words, max_blocks, page, nq, nkv, window, splits, B, tokens, num_pages, scale, cap};
  if (part != nullptr) p.part_ml = part + (size_t)tokens * nq * splits * D;
  return bf16 ? run_rows<__nv_bfloat16>(p, B, max_t, (cudaStream_t)stream) : run_rows<float>(p, B, max_t, (cudaStream_t)stream);
}
