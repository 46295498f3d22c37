// Attention of a tree of drafted tokens over the paged cache.
//
// Compiled once per head size: -DTS_HEAD_DIM=<multiple of 8, at most 256>.
//
// A request brings t tokens to a step, the nodes of a tree, and has n rows in the cache, the last t of them its nodes'.  Node i sees every row j < n - t
// (with a window: those with j > pos_i - window) and, of the step's rows, row n - t + k where bit k of its mask is set (with a window: and pos_k > pos_i - window).
//   o_i = sum_j p_ij v_j,  p_i = softmax over the rows it sees (and its head's sink) of s_ij = scale q_i k_j, or cap tanh(scale q_i k_j / cap).
// A node that sees nothing gets zeros.  Scores, maxima, sums and outputs are float32 until the end.
//
// This file takes float32 and the heads that attention_tree_tcgen05.cu does not.  The (node, query head of a group) pairs of a request are the rows of a tile for
// each KV head, so that what is read of the cache is read once for them all; the keys are cut into parts, a CTA each, whose results (maximum, sum, unnormalised
// output) a second kernel joins, always in the same order.
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

// Whether the token (global number `token`, position `pos`) of a request whose nodes begin at token q_begin and at row `first` sees row j of n.
__device__ __forceinline__ bool sees(const Params& p, int token, int pos, int j, int n, int first, int q_begin) {
  if (j >= n) return false;
  const int node = j - first;
  if (node < 0) return p.window == 0 || j > pos - p.window;
  if ((node >> 6) >= p.words || !((p.mask[(size_t)token * p.words + (node >> 6)] >> (node & 63)) & 1)) return false;
  return p.window == 0 || p.positions[q_begin + node] > pos - p.window;
}

// ---------------------------------------------------------------------------
// mma.sync: 16 WM rows, of which every warp holds 16, against blocks of keys, cut among 8 / WM warps; a warp walks its keys with maxima and sums of its own, and the
// CTA joins its warps at the end.  bfloat16: products as they are, weights rounded to bfloat16 (their values' type).  float32: every operand is the sum of
// two tf32 (11 bits each), a product three: h h' + h l' + l h'; what is left out is below 2^-21 of it, where a float32 sum is off by 2^-24 a
// term.
//
// The order of the entries inside a product does not matter, and the order of columns of the result is put right at the end: a lane takes 16 neighbouring bytes of
// a row of queries or keys as its share of two products (for float32 values: four neighbouring columns of a row as its share of four), one load without conflicts.
//
// What bounds it: the old path of the tensor cores, where any such product takes 8 cycles (three of 16 x 8 x 8 a term in float32: 90 TFLOP/s of whole terms a GPU) and
// other arithmetic hardly runs beside it.  16 requests of 2,000 rows, 32 nodes, float32: 366 us (45 TFLOP/s), the rest cuts operands in two; 8 of 4,000, 64 nodes, bfloat16 heads of
// 256: 293 (226 TFLOP/s), the rest are loads from shared memory (as many cycles as the products) and weights.  Few rows are bound by the copies: chains of 4 over
// 4,000 rows, heads of 256, 63 us (4.2 TB/s).

constexpr int TH = 256;

template <typename T, int WM>
struct Tile {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int WN = 8 / WM;                                 // warps that share a block's keys
  static constexpr int BN = !F32 && WN == 8 ? 128 : 64;             // keys of a block (a warp's at least a product's: 8 in float32, 16 in bfloat16)
  static constexpr int RM = 16 * WM;
  static constexpr int NT = BN / WN / 8;                            // 8s of keys per warp
  static constexpr int CHUNK = 64 / sizeof(T);                      // columns that four lanes take at a time
  static constexpr int DK = (D + CHUNK - 1) / CHUNK * CHUNK;        // columns of queries and keys, zeros behind D
  static constexpr int KB = DK * sizeof(T);                         // bytes of such a row
  static constexpr int FLIP = KB % 128 == 0 ? 64 : 0;               // its halves of 128 bytes change places in odd rows: 64 bytes of two rows lie in different banks
  static constexpr int DV = F32 ? (D + 31) / 32 * 32 : (D + 15) / 16 * 16;  // columns of values (what stands behind D goes to columns that nobody reads)
  static constexpr int VB = DV * sizeof(T) + 16;
  static constexpr int OT = DV / 8;
  static constexpr int OUT = 8 * 16 * DV * 4;                       // the warps' results, when all else has been read
  static constexpr int STAGE = BN * (KB + VB);
  // Heads up to 64: two CTAs on an SM, a block each in shared memory (12 requests with a window of 1,024, 13 nodes, float32: two blocks each 3 % slower).  Larger
  // ones: one CTA, and two blocks where they find room, the next one's copies asked for between the products of this one (8 of 4,000 rows, 16 nodes, bfloat16 heads
  // of 256: with one block 17 % slower).
  static constexpr int CTAS = D <= 64 ? 2 : 1, ROOM = CTAS == 2 ? 112 * 1024 : 226 * 1024;
  static constexpr int STAGES = CTAS == 1 && RM * KB + 2 * STAGE <= ROOM ? 2 : 1;
  static constexpr int K_AT = RM * KB, V_AT = K_AT + BN * KB, END = K_AT + STAGES * STAGE;
  static constexpr int SMEM = END > OUT ? END : OUT;
  static_assert(SMEM <= ROOM, "shared memory of an SM");
};

__device__ __forceinline__ void copy16(unsigned char* dst, const void* src, bool there) {
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
  const int bytes = there ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void rows_landed() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
  __syncthreads();
}

__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&x)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
}
// x as the sum of two tf32: the upper rounded to nearest, the lower the rest, of which a product reads the upper 19 bits (11 significant ones; with it rounded, too, two
// more instructions an operand).  Bits of an infinity stay; a NaN stays in the lower part at the least.
__device__ __forceinline__ void cut(uint32_t x, uint32_t& high, uint32_t& low) {
  high = (x + 0x1000u) & 0xffffe000u;
  low = __float_as_uint(__uint_as_float(x) - __uint_as_float(high));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float power2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh; on bfloat16 as 1 - 2 / (e^2x + 1), exact at both ends, off by a few 1e-7 in between (the weights' own rounding is 2^-9).
template <bool ACCURATE>
__device__ __forceinline__ float bent(float x) {
  return ACCURATE ? tanhf(x) : 1.f - __fdividef(2.f, __expf(2.f * x) + 1.f);
}
// The lowest and the highest position of a request's nodes (with a window), by every warp for itself.
__device__ __forceinline__ int2 position_range(const Params& p, int q_begin, int t) {
  int lowest = INT_MAX, highest = INT_MIN;
  for (int i = threadIdx.x & 31; i < t; i += 32) {
    const int x = p.positions[q_begin + i];
    lowest = min(lowest, x), highest = max(highest, x);
  }
  return make_int2(__reduce_min_sync(0xffffffffu, lowest), __reduce_max_sync(0xffffffffu, highest));
}

template <typename T, int WM>
__global__ void __launch_bounds__(TH, Tile<T, WM>::CTAS) tree_rows_kernel(const Params p) {
  ts_pdl_prologue();
  using L = Tile<T, WM>;
  constexpr bool F32 = L::F32;
  constexpr int BN = L::BN, RM = L::RM, NT = L::NT, WN = L::WN, CHUNKS = L::KB / 64, LINES = (D * (int)sizeof(T) + 127) / 128, COPIES = BN / 32;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float2 ml_s[8][16];
  unsigned char *Qs = smem, *Ks = smem + L::K_AT, *Vs = smem + L::V_AT;
  const int split = blockIdx.x, hk = blockIdx.y % p.nkv, tile = blockIdx.y / p.nkv, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int wm = warp / WN, wn = warp % WN;
  const int q_begin = p.cu[b], t = p.cu[b + 1] - q_begin, n = p.context[b], first = n - t;
  const int G = p.nq / p.nkv, rows = t * G, r0 = tile * RM;
  if (t <= 0 || r0 >= rows) return;
  // the first row that any node sees, and the row from which on a window hides nothing of what is before the step
  int lo = 0, whole_from = 0;
  if (p.window > 0) {
    const int2 range = position_range(p, q_begin, t);
    const long long from = (long long)range.x - p.window + 1;
    lo = (int)(from < 0 ? 0 : from > first ? max(first, 0) : from);
    whole_from = max(range.y - p.window + 1, 0);
  }
  // this CTA's blocks of keys: an even share of the request's
  const int kb0 = lo / BN, blocks = n > 0 ? (n - 1) / BN - kb0 + 1 : 0;
  const int per = (blocks + p.splits - 1) / p.splits, begin = kb0 + split * per, end = min(kb0 + blocks, begin + per);
  const int* table = p.table + (size_t)b * p.max_blocks;
  // A thread copies an eighth of every 128 bytes of the rows tid / 8, tid / 8 + 32, ...  Where they begin in the pool: their pages are asked for a block ahead.
  int page[COPIES], in_page[COPIES];
  long long at[COPIES];
  auto ask_page = [&](int blk) {
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int j = blk * BN + tid / 8 + 32 * i, e = j / p.page;
      page[i] = -1, in_page[i] = j - e * p.page;
      if (blk < end && j < n && e < p.max_blocks) page[i] = table[e];
    }
  };
  auto find_rows = [&]() {
#pragma unroll
    for (int i = 0; i < COPIES; ++i) at[i] = page[i] >= 0 && page[i] < p.num_pages ? ((((long long)page[i] * p.page + in_page[i]) * p.nkv + hk) * D) * (long long)sizeof(T) : -1;
  };
  auto copy_keys = [&](int c, int stage) {
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int row = tid / 8 + 32 * i, from = c * 128 + (tid & 7) * 16;
      if (D * sizeof(T) % 128 == 0 || from < D * (int)sizeof(T))
        copy16(Ks + stage * L::STAGE + row * L::KB + (from ^ (row & 1) * L::FLIP), static_cast<const unsigned char*>(p.k) + (at[i] < 0 ? 0 : at[i] + from), at[i] >= 0);
    }
  };
  auto copy_values = [&](int c, int stage) {
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int row = tid / 8 + 32 * i, from = c * 128 + (tid & 7) * 16;
      if (D * sizeof(T) % 128 == 0 || from < D * (int)sizeof(T))
        copy16(Vs + stage * L::STAGE + row * L::VB + from, static_cast<const unsigned char*>(p.v) + (at[i] < 0 ? 0 : at[i] + from), at[i] >= 0);
    }
  };
  if (begin < end) {
    ask_page(begin);
    // queries: row r of the tile is token r / G, head r % G; zeros behind the rows and the columns.  (Entry by entry they took as long as two blocks: 8 requests of
    // 4,000 rows, 64 nodes, heads of 256 362 us, with copies of 16 bytes 293.)
    if (((uintptr_t)p.q & 15) == 0) {
#pragma unroll 4
      for (int i = tid; i < RM * (L::KB / 16); i += TH) {
        const int x = i / (L::KB / 16), r = r0 + x, from = i % (L::KB / 16) * 16;
        const bool there = r < rows && from < D * (int)sizeof(T);
        copy16(Qs + x * L::KB + (from ^ (x & 1) * L::FLIP),
               static_cast<const unsigned char*>(p.q) + (there ? ((size_t)(q_begin + r / G) * p.nq + hk * G + r % G) * D * sizeof(T) + from : 0), there);
      }
    } else {
      const T* q = reinterpret_cast<const T*>(p.q);
      for (int i = tid; i < RM * L::DK; i += TH) {
        const int x = i / L::DK, r = r0 + x, c = i % L::DK;
        *reinterpret_cast<T*>(Qs + x * L::KB + ((c * (int)sizeof(T)) ^ (x & 1) * L::FLIP)) =
            r < rows && c < D ? q[((size_t)(q_begin + r / G) * p.nq + hk * G + r % G) * D + c] : ts_from_float<T>(0.f);
      }
    }
    find_rows();
    ask_page(begin + 1);
#pragma unroll 4
    for (int c = 0; c < LINES; ++c) copy_keys(c, 0);
    if (L::STAGES == 1) copies_end();
#pragma unroll 4
    for (int c = 0; c < LINES; ++c) copy_values(c, 0);
    copies_end();
  }
  if constexpr (L::DK > D) {  // (a product with zeros needs numbers beside them)
    constexpr int PAD = L::DK - D;
    for (int i = tid; i < L::STAGES * BN * PAD; i += TH) {
      const int x = i / PAD % BN, c = (D + i % PAD) * (int)sizeof(T);
      *reinterpret_cast<T*>(Ks + i / (BN * PAD) * L::STAGE + x * L::KB + (c ^ (x & 1) * L::FLIP)) = ts_from_float<T>(0.f);
    }
  }
  const bool works = r0 + wm * 16 < rows;
  int token[2], pos[2];
  float m[2], l[2], o[L::OT][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + wm * 16 + g + 8 * h;
    token[h] = r < rows ? q_begin + r / G : -1;
    pos[h] = token[h] >= 0 && p.window > 0 ? p.positions[token[h]] : 0;
    m[h] = -INFINITY, l[h] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < L::OT; ++i)
#pragma unroll
    for (int x = 0; x < 4; ++x) o[i][x] = 0.f;
  // scores in units of log2, what enters 2^x: a product times `scale`, or cap_log2 times the tanh of that
  const float scale = p.cap > 0.f ? p.scale / p.cap : p.scale * LOG2E, cap_log2 = p.cap * LOG2E;
  const unsigned char *q_row = Qs + (wm * 16 + g) * L::KB + t4 * 16, *k_row = Ks + (wn * NT * 8 + g) * L::KB + t4 * 16;
  const int flip = (g & 1) * L::FLIP;
#pragma unroll 1
  for (int blk = begin; blk < end; ++blk) {
    const bool more = blk + 1 < end;
    const int stage = L::STAGES == 2 ? (blk - begin) & 1 : 0;
    if (more) find_rows(), ask_page(blk + 2);
    rows_landed<L::STAGES == 2 ? 0 : 1>();
    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[j][x] = 0.f;
    if (works) {
      // Keys in groups, a chunk of columns a time; the next block's copies go out during the first group.  In float32 a chunk's products are summed from zero and
      // then added: a tensor core cuts its sums off instead of rounding them, and along whole rows and blocks that was ten times the error of a float32 sum (12 requests
      // with a window of 1,024: 3.1e-6 relative to 64 bits, 2.4e-7 so, plain float32 6.7e-7; 85 us, 92 so).
      constexpr int J = F32 && NT > 4 ? 4 : NT;
#pragma unroll
      for (int j0 = 0; j0 < NT; j0 += J) {
#pragma unroll 2
        for (int c = 0; c < CHUNKS; ++c) {
          if (L::STAGES == 2 && j0 == 0 && more && c % 2 == 0) copy_keys(c / 2, stage ^ 1), copy_values(c / 2, stage ^ 1);
          const int here = (c * 64) ^ flip;
          const uint4 a = *reinterpret_cast<const uint4*>(q_row + here), a8 = *reinterpret_cast<const uint4*>(q_row + 8 * L::KB + here);
          const unsigned char* keys = k_row + stage * L::STAGE + here + j0 * 8 * L::KB;
          uint4 k[J];
#pragma unroll
          for (int j = 0; j < J; ++j) k[j] = *reinterpret_cast<const uint4*>(keys + j * 8 * L::KB);
          // (a product waits for the one before it on the same scores: those of several keys take turns)
          if constexpr (F32) {
            uint32_t ah[8], al[8], kh[J][4], kl[J][4];
            cut(a.x, ah[0], al[0]), cut(a8.x, ah[1], al[1]), cut(a.y, ah[2], al[2]), cut(a8.y, ah[3], al[3]);
            cut(a.z, ah[4], al[4]), cut(a8.z, ah[5], al[5]), cut(a.w, ah[6], al[6]), cut(a8.w, ah[7], al[7]);
#pragma unroll
            for (int j = 0; j < J; ++j) cut(k[j].x, kh[j][0], kl[j][0]), cut(k[j].y, kh[j][1], kl[j][1]), cut(k[j].z, kh[j][2], kl[j][2]), cut(k[j].w, kh[j][3], kl[j][3]);
            float x[J][4];
#pragma unroll
            for (int j = 0; j < J; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
              for (int j = 0; j < J; ++j) mma_tf32(x[j], al[4 * u], al[4 * u + 1], al[4 * u + 2], al[4 * u + 3], kh[j][2 * u], kh[j][2 * u + 1]);
#pragma unroll
              for (int j = 0; j < J; ++j) mma_tf32(x[j], ah[4 * u], ah[4 * u + 1], ah[4 * u + 2], ah[4 * u + 3], kl[j][2 * u], kl[j][2 * u + 1]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int j = 0; j < J; ++j) mma_tf32(x[j], ah[4 * u], ah[4 * u + 1], ah[4 * u + 2], ah[4 * u + 3], kh[j][2 * u], kh[j][2 * u + 1]);
#pragma unroll
            for (int j = 0; j < J; ++j) s[j0 + j][0] += x[j][0], s[j0 + j][1] += x[j][1], s[j0 + j][2] += x[j][2], s[j0 + j][3] += x[j][3];
          } else {
#pragma unroll
            for (int j = 0; j < J; ++j) mma_bf16(s[j], a.x, a8.x, a.y, a8.y, k[j].x, k[j].y);
#pragma unroll
            for (int j = 0; j < J; ++j) mma_bf16(s[j], a.z, a8.z, a.w, a8.w, k[j].z, k[j].w);
          }
        }
      }
    }
    if (L::STAGES == 2) {
      if (!works && more)
        for (int c = 0; c < LINES; ++c) copy_keys(c, stage ^ 1), copy_values(c, stage ^ 1);
      copies_end();
    } else {
      __syncthreads();  // the keys have been read
#pragma unroll 4
      for (int c = 0; c < LINES && more; ++c) copy_keys(c, 0);
      copies_end();
    }
    if (works) {
      // seen by every token: rows before the step that no window hides
      const bool open = blk * BN + BN <= first && blk * BN >= whole_from;
      const int key0 = blk * BN + wn * NT * 8 + 2 * t4;
      if (p.cap > 0.f) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[j][x] = cap_log2 * bent<F32>(s[j][x] * scale);
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[j][x] *= scale;
      }
      if (!open) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (token[x >> 1] < 0 || !sees(p, token[x >> 1], pos[x >> 1], key0 + 8 * j + (x & 1), n, first, q_begin)) s[j][x] = -INFINITY;
      }
      float corr[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NT; ++j) top = fmaxf(top, fmaxf(s[j][2 * h], s[j][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m_new = fmaxf(m[h], top), off = m_new == -INFINITY ? 0.f : m_new;
        corr[h] = power2(m[h] - off);
        m[h] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float& v = s[j][2 * h + x];
            v = power2(v - off);
            sum += v;
          }
        l[h] = l[h] * corr[h] + sum;  // (of this lane's keys)
      }
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < L::OT; ++i) o[i][0] *= corr[0], o[i][1] *= corr[0], o[i][2] *= corr[1], o[i][3] *= corr[1];
      }
    }
    if (L::STAGES == 1) rows_landed<1>();
    if (works) {
      if constexpr (F32) {
        constexpr int J = NT > 1 && D <= 128 ? 2 : 1;  // 8s of keys whose products are summed from zero and then added
#pragma unroll
        for (int j0 = 0; j0 < NT; j0 += J) {
          uint32_t ph[J][4], pl[J][4];  // (the product's key t is this lane's first, t + 4 its second)
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const float* w = s[j0 + j];
            cut(__float_as_uint(w[0]), ph[j][0], pl[j][0]), cut(__float_as_uint(w[2]), ph[j][1], pl[j][1]);
            cut(__float_as_uint(w[1]), ph[j][2], pl[j][2]), cut(__float_as_uint(w[3]), ph[j][3], pl[j][3]);
          }
          const unsigned char* row = Vs + stage * L::STAGE + (wn * NT * 8 + 8 * j0 + 2 * t4) * L::VB + g * 16;
#pragma unroll
          for (int c = 0; c < L::DV / 32; ++c) {
            uint32_t h[J][4][2], l[J][4][2];
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(row + (8 * j + i) * L::VB + c * 128);
                cut(v.x, h[j][0][i], l[j][0][i]), cut(v.y, h[j][1][i], l[j][1][i]), cut(v.z, h[j][2][i], l[j][2][i]), cut(v.w, h[j][3][i], l[j][3][i]);
              }
            float x[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j) {
#pragma unroll
              for (int i = 0; i < 4; ++i) mma_tf32(x[i], pl[j][0], pl[j][1], pl[j][2], pl[j][3], h[j][i][0], h[j][i][1]);
#pragma unroll
              for (int i = 0; i < 4; ++i) mma_tf32(x[i], ph[j][0], ph[j][1], ph[j][2], ph[j][3], l[j][i][0], l[j][i][1]);
            }
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) mma_tf32(x[i], ph[j][0], ph[j][1], ph[j][2], ph[j][3], h[j][i][0], h[j][i][1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[4 * c + i][0] += x[i][0], o[4 * c + i][1] += x[i][1], o[4 * c + i][2] += x[i][2], o[4 * c + i][3] += x[i][3];
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j + 1 < NT; j += 2) {
          const uint32_t p0 = pack_bf16(s[j][0], s[j][1]), p1 = pack_bf16(s[j][2], s[j][3]), p2 = pack_bf16(s[j + 1][0], s[j + 1][1]), p3 = pack_bf16(s[j + 1][2], s[j + 1][3]);
          const uint32_t row = (uint32_t)__cvta_generic_to_shared(Vs + stage * L::STAGE + (wn * NT * 8 + 8 * j + (lane & 15)) * L::VB + (lane >> 4) * 16);
          // (asked for two products ahead)
          uint32_t x[2][4];
          ldmatrix4(x[0], row);
#pragma unroll
          for (int c = 0; c < L::DV / 16; ++c) {
            if (c + 1 < L::DV / 16) ldmatrix4(x[(c + 1) & 1], row + (c + 1) * 32);
            mma_bf16(o[2 * c], p0, p1, p2, p3, x[c & 1][0], x[c & 1][1]);
            mma_bf16(o[2 * c + 1], p0, p1, p2, p3, x[c & 1][2], x[c & 1][3]);
          }
        }
      }
    }
    if (L::STAGES == 1) {
      __syncthreads();  // the values have been read
#pragma unroll 4
      for (int c = 0; c < LINES && more; ++c) copy_values(c, 0);
      copies_end();
    }
  }
  __syncthreads();  // (queries, too: the results go over all of them)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (t4 == 0) ml_s[warp][g + 8 * h] = make_float2(m[h], l[h]);
    float* mine = reinterpret_cast<float*>(smem) + (warp * 16 + g + 8 * h) * L::DV;
    if constexpr (F32) {
#pragma unroll
      for (int c = 0; c < L::DV / 32; ++c) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *reinterpret_cast<float4*>(mine + 32 * c + 8 * t4 + 4 * x) = make_float4(o[4 * c][2 * h + x], o[4 * c + 1][2 * h + x], o[4 * c + 2][2 * h + x], o[4 * c + 3][2 * h + x]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < L::OT; ++i) *reinterpret_cast<float2*>(mine + 8 * i + 2 * t4) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
    }
  }
  __syncthreads();
  // the warps of a row, joined in one order, four columns a thread
  for (int i = tid; i < RM * (D / 4); i += TH) {
    const int x = i / (D / 4), c = i % (D / 4) * 4, r = r0 + x;
    if (r >= rows) break;
    const int w0 = x / 16 * WN, head = hk * G + r % G;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WN; ++w) top = fmaxf(top, ml_s[w0 + w][x % 16].x);
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WN; ++w) {
      const float2 ml = ml_s[w0 + w][x % 16];
      const float f = ml.x == -INFINITY ? 0.f : power2(ml.x - top);
      const float4 z = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) + ((w0 + w) * 16 + x % 16) * L::DV + c);
      sum += f * ml.y;
      if (f > 0.f) y.x = fmaf(f, z.x, y.x), y.y = fmaf(f, z.y, y.y), y.z = fmaf(f, z.z, y.z), y.w = fmaf(f, z.w, y.w);
    }
    const size_t row = (size_t)(q_begin + r / G) * p.nq + head;
    if (p.splits > 1) {
      const size_t at = row * p.splits + split;
      if (c == 0) p.part_ml[2 * at] = top, p.part_ml[2 * at + 1] = sum;
      *reinterpret_cast<float4*>(p.part_o + at * D + c) = y;
    } else {
      float f = 1.f;
      if (p.head_sinks != nullptr) {
        const float sink = p.head_sinks[head] * LOG2E, over = fmaxf(top, sink);
        f = top == -INFINITY ? 0.f : exp2f(top - over);
        sum = sum * f + (sink == -INFINITY ? 0.f : exp2f(sink - over));
      }
      const float inv = sum > 0.f ? f / sum : 0.f;
      T* out = reinterpret_cast<T*>(p.out) + row * D + c;
      out[0] = ts_from_float<T>(y.x * inv), out[1] = ts_from_float<T>(y.y * inv), out[2] = ts_from_float<T>(y.z * inv), out[3] = ts_from_float<T>(y.w * inv);
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

template <typename T, int WM>
int launch_rows(const Params& p, int B, int rows, cudaStream_t stream) {
  using L = Tile<T, WM>;
  const int tiles = (rows + L::RM - 1) / L::RM;
  if ((long long)tiles * p.nkv > 65535 || B > 65535) return TS_ERR_UNSUPPORTED_SIZE;
  const cudaError_t e = cudaFuncSetAttribute(tree_rows_kernel<T, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  if (e != cudaSuccess) return (int)e;
  return ts_launch(tree_rows_kernel<T, WM>, dim3(p.splits, tiles * p.nkv, B), dim3(TH), L::SMEM, stream, p);
}

// Warps beside one another by the rows of the largest request: the fewest that hold them all.  Many rows take eight (four in float32 and heads above 128, which
// leave no room beside the keys for more), unless that would leave half of the last tile empty (16 requests of 2,000 rows, 33 nodes of four heads, float32: eight
// 723 us, four 516; 48 nodes 724 and 589; bfloat16 heads of 256, 33 nodes 291 and 271).
template <typename T>
constexpr int most_warps() { return sizeof(T) == 4 && D > 128 ? 4 : 8; }
template <typename T>
int warps_beside(int rows) {
  if (rows <= 64) return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  return rows > 128 && rows % 128 > 0 && rows % 128 <= 64 ? 4 : most_warps<T>();
}

template <typename T>
int run_rows(const Params& p, int B, int max_t, cudaStream_t stream) {
  const int rows = max_t * (p.nq / p.nkv), wm = warps_beside<T>(rows);
  const int status = wm == 1 ? launch_rows<T, 1>(p, B, rows, stream) : wm == 2 ? launch_rows<T, 2>(p, B, rows, stream)
                     : wm == 4 ? launch_rows<T, 4>(p, B, rows, stream) : launch_rows<T, most_warps<T>()>(p, B, rows, stream);
  if (status != 0 || p.splits == 1) return status;
  return ts_launch(join_parts_kernel<T>, dim3(((size_t)p.tokens * p.nq + 3) / 4), dim3(128), 0, stream, p);
}

template <typename T, int WM>
void sizes_of(int& rm, int& bn, int& ctas) { rm = Tile<T, WM>::RM, bn = Tile<T, WM>::BN, ctas = Tile<T, WM>::CTAS; }

template <typename T>
int splits_of(int B, int rows, int nkv, int max_context) {
  const int wm = warps_beside<T>(rows);
  int rm, bn, ctas;
  wm == 1 ? sizes_of<T, 1>(rm, bn, ctas) : wm == 2 ? sizes_of<T, 2>(rm, bn, ctas) : wm == 4 ? sizes_of<T, 4>(rm, bn, ctas) : sizes_of<T, most_warps<T>()>(rm, bn, ctas);
  const long long units = (long long)B * nkv * ((rows + rm - 1) / rm), slots = 148ll * ctas;
  const int blocks = (max_context + bn - 1) / bn;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 64 && s <= (blocks < 1 ? 1 : blocks); ++s) {
    const double cost = (double)((units * s + slots - 1) / slots) * ((blocks + s - 1) / s + 1.5);
    if (s == 1 || cost < 0.98 * least) best = s, least = cost;
  }
  return best;
}

}  // namespace

// In how many parts the keys of a request of `max_context` rows are cut: the fewest blocks in a row, counting every wave of CTAs (as many as
// registers and shared memory let run at once) and one and a half blocks for a CTA's start and the joining of its part.
TS_EXPORT int ts_attention_tree_splits(int bf16, int B, int max_t, int nq, int nkv, int max_context) {
  const int rows = max_t * (nq / nkv);
  return bf16 ? splits_of<__nv_bfloat16>(B, rows, nkv, max_context) : splits_of<float>(B, rows, nkv, max_context);
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
