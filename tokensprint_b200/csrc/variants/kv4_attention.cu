// Causal attention over a cache held in 4 bits, and the weight that it gives to every cached row, for one
// head size (-DTS_HEAD_DIM=64, 128 or 256).
//
// For the rows r of a tile (query token i, query head of the key head's group) and the keys j that i may see:
//   s_rj = scale q_r . k_j      o_r = sum_j p_rj v_j      p_rj = exp(s_rj - m_r) / l_r      l_r = sum_j exp(s_rj - m_r) (+ exp(sink - m_r))
// with the running maximum m and sum l of one pass over the keys, in 32 bits.  The matrix instructions take bfloat16: keys
// and values in 4 bits are exact in it, and so are queries of that type.  exp(s - m) is given as two of them (16 bits; one has 8,
// and half, with 11, loses weights below 2^-24 of the largest), float32 queries and their weights as three.
//
// Keys stand on the M side of the instruction: S^T[16 keys][8 rows] = K Q^T and O^T[channels][8 rows] += V^T P^T, so
// that the few rows of a decode step fill an instruction and every code is unpacked once for all of them.
//
// What bounds it: for 4 query rows a key head a record of 16 tokens (2,304 bytes with heads of 128) takes a warp some 400 instructions (the codes
// of 4,096 values unpacked two at a time: a shift, a mask and an or in one, a multiply-add; 16 products; the softmax), and the pipes that
// run them (integer 54 % busy, multiply-add 37 %, tensor 20 %) share the issue slots: 3.5 TB/s of cache where the same kernel without the arithmetic
// reads 5.8.  tcgen05 does not fit: its smallest tile is 128 keys by 8 rows whose operands must lie unpacked in shared memory or tensor memory, so
// every value would be written and read once more, and unpacking is what the time goes into.  us with 32 query and 8 key heads of 128:
// 4 requests of up to 60,000 rows 78 (276 MB), 32 of up to 4,096 36 (96 MB), 1 of 517 (16 query heads) 10.4.
#include "kv4.cuh"

#ifndef TS_HEAD_DIM
#error "compile with -DTS_HEAD_DIM=64, 128 or 256"
#endif

namespace {

constexpr int D = TS_HEAD_DIM;
using Rec = Kv4Record<D>;
constexpr int kWarps = 4;
constexpr int kRing = 4;  // records of a warp's ring
constexpr float kLowest = -3.402823466e38f;  // the running maximum before the first key (finite: no difference of it is NaN)
constexpr int kMaxTiles = 1024;  // (sequence, row tile) pairs of a launch: a CTA keeps their key ranges in shared memory
constexpr int kMaxParts = 64;    // most CTAs that share a key range
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  const void* q;
  const uint8_t* pool;
  void* out;
  float* lse;
  const float* sinks;
  const int* cu;
  const int* context;
  const int* table;
  float* part;
  int* tickets;
  int table_stride, page_blocks, num_pages, tokens, num_seqs, nq, nkv, group, window, row_tiles, first_tile;
  float scale;  // times log2 e
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src));
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The record of block `blk` of a request, given its entry of the block table.
__device__ __forceinline__ const uint8_t* record(const Params& p, int page, int blk, int head) {
  return p.pool + (((size_t)min(max(page, 0), p.num_pages - 1) * p.nkv + head) * p.page_blocks + blk % p.page_blocks) * Rec::kBytes;
}

// O^T[channels][rows] += V^T P^T of one record.  Lane (g, t) owns the channels [g D/8, (g+1) D/8) and reads of them the
// tokens 2t, 2t+1, 2t+8, 2t+9; p[tile][part]: the transposed weights of tokens 0..7 and 8..15.  Tokens outside
// [first, last) count as zeros, whatever the record holds there.
template <int kTiles, int kP, bool kEdge>
__device__ __forceinline__ void add_values(const uint8_t* rec, const uint32_t (&p)[kTiles][kP][2], float (&o)[kTiles][D / 16][4], int g, int t,
                                           int first, int last) {
  constexpr int kWords = D / 64;
  const uint8_t* codes = rec + Rec::kValues + g * (D / 16);
  const uint8_t* scales = rec + Rec::kValueScales + g * kWords / 2;  // (heads of 64: two lanes share a group)
  uint32_t w[4][kWords], sc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int token = 2 * t + (i & 1) + 8 * (i >> 1);
    const uint8_t* c = codes + token * (D / 2);
    if constexpr (kWords == 1) w[i][0] = *reinterpret_cast<const uint32_t*>(c);
    else if constexpr (kWords == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(c);
      w[i][0] = v.x, w[i][1] = v.y;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(c);
      w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
    }
    if constexpr (kWords == 4) sc[i] = *reinterpret_cast<const uint16_t*>(scales + token * (D / 16));
    else sc[i] = scales[token * (D / 16)];
    if (kEdge && (token < first || token >= last)) sc[i] = 0;
  }
#pragma unroll
  for (int grp = 0; grp < (kWords + 1) / 2; ++grp) {
    __nv_bfloat162 f[2], c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) kv4_factors((sc[2 * i] >> (8 * grp)) & 0xffu, (sc[2 * i + 1] >> (8 * grp)) & 0xffu, f[i], c[i]);
#pragma unroll
    for (int k = 2 * grp; k < (kWords == 1 ? 1 : 2 * grp + 2); ++k) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // four channels each: 8k + 4 half + 0..3
        const uint32_t sel = half ? 0x7632u : 0x5410u;
        const uint32_t x = __byte_perm(w[0][k], w[1][k], sel), y = __byte_perm(w[2][k], w[3][k], sel);
        const uint32_t a0 = kv4_pair(x << 3, f[0], c[0]), a1 = kv4_pair(x >> 1, f[0], c[0]);
        const uint32_t a2 = kv4_pair(y << 3, f[1], c[1]), a3 = kv4_pair(y >> 1, f[1], c[1]);
        const uint32_t b0 = kv4_pair(x >> 5, f[0], c[0]), b1 = kv4_pair(x >> 9, f[0], c[0]);
        const uint32_t b2 = kv4_pair(y >> 5, f[1], c[1]), b3 = kv4_pair(y >> 9, f[1], c[1]);
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int part = 0; part < kP; ++part) {
            kv4_mma(o[n][4 * k + 2 * half], a0, a1, a2, a3, p[n][part][0], p[n][part][1]);
            kv4_mma(o[n][4 * k + 2 * half + 1], b0, b1, b2, b3, p[n][part][0], p[n][part][1]);
          }
      }
    }
  }
}

// What a tile of rows of one sequence and key head is, and which rows it holds.
struct Tile {
  int b, head, first_row, rows, q_start, q_len, context;
  // (lengths are kept within the block table and the tensors, so that no wrong number reads beyond them)
  __device__ __forceinline__ void open(const Params& p, int seq, int key_head) {
    b = seq, head = key_head;
    q_start = min(max(p.cu[b], 0), p.tokens);
    q_len = min(max(p.cu[b + 1], q_start), p.tokens) - q_start;
    context = min(p.context[b], p.table_stride * p.page_blocks * KV4_BLOCK);
    rows = q_len * p.group;
  }
  __device__ __forceinline__ int position(const Params& p, int row) const { return context - q_len + row / p.group; }  // the last key it sees
  __device__ __forceinline__ int token(const Params& p, int row) const { return q_start + row / p.group; }
  template <typename T>
  __device__ __forceinline__ const T* query(const Params& p, int row) const {
    return reinterpret_cast<const T*>(p.q) + ((size_t)token(p, row) * p.nq + query_head(p, row)) * D;
  }
  __device__ __forceinline__ int query_head(const Params& p, int row) const { return head * p.group + row % p.group; }
};

// A finished row: o over its sum l of 2^(s - m), with the sink's share.
template <typename T>
__device__ __forceinline__ void write_row(const Params& p, const Tile& tile, int row, int channel, float4 o, float m, float l) {
  const int head = tile.query_head(p, row);
  if (p.sinks != nullptr) {
    const float sink = p.sinks[head] * kLog2e, top = fmaxf(m, sink), f = kv4_exp2(m - top);  // (m is finite, so a sink of -inf is none)
    l = l * f + kv4_exp2(sink - top);
    o.x *= f, o.y *= f, o.z *= f, o.w *= f;
    m = top;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
  const size_t at = ((size_t)tile.token(p, row) * p.nq + head) * D + channel;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  } else {
    __nv_bfloat162 v[2] = {__floats2bfloat162_rn(o.x * inv, o.y * inv), __floats2bfloat162_rn(o.z * inv, o.w * inv)};
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + at) = *reinterpret_cast<const uint2*>(v);
  }
  if (p.lse != nullptr && channel == 0) p.lse[(size_t)tile.token(p, row) * p.nq + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Parts of one row (maximum, sum, four channels) added to one another.
struct RowSum {
  float m = kLowest, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float pm, float pl, float4 v, float top) {
    const float f = kv4_exp2(pm - top);
    l += f * pl;
    o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
  }
};

// The key ranges of all (sequence, row tile) pairs, counted in steps of kRecords records, one behind the other; every key head has them again.
// A CTA's share is an equal part of all of them, whatever the lengths are, and may begin and end inside a range.
struct Shares {
  int* before;  // [pairs + 1]: steps of one head before the pair
};

template <typename T, int kTiles, int kQ, int kP, int kRecords, bool kTwice>
__global__ void __launch_bounds__(kWarps * 32, D > 128 || sizeof(T) != 2 ? 1 : kTiles == 1 ? 4 : 3) attention_kernel(const Params p) {
  // kTwice: a tile of 4 rows, which stand twice among the 8 columns; the first time with the first part of their weights, the second time
  // with the second, so that one product adds both (of 24 products a record 16 are left).
  static_assert(!kTwice || (kTiles == 1 && kP == 2), "four rows, two parts");
  constexpr int kRows = kTwice ? 4 : 8 * kTiles, kParts = kTwice ? 1 : kP, kColumnRows = kTwice ? 4 : 8;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int scratch[kWarps + 2];
  ts_pdl_prologue();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int pairs = p.num_seqs * p.row_tiles;
  uint4* sq = reinterpret_cast<uint4*>(smem + kWarps * kRing * Rec::kBytes);  // the queries: [tiles][parts][words][lanes]
  float* so = reinterpret_cast<float*>(sq + kTiles * kQ * D);                 // the warps' parts: [warps][rows][D]
  float* sm = so + kWarps * kRows * D;                                        // [warps][rows]
  float* sl = sm + kWarps * kRows;
  const Shares shares = {reinterpret_cast<int*>(sl + kWarps * kRows)};

  auto open = [&](Tile& tile, int pair, int head) {
    tile.open(p, pair / p.row_tiles, head);
    tile.first_row = (p.first_tile + pair % p.row_tiles) * kRows;
  };
  auto first_record = [&](const Tile& tile) { return p.window > 0 ? max(0, tile.position(p, tile.first_row) - p.window + 1) / KV4_BLOCK : 0; };
  // ---- the shares: a block-wide sum over the pairs, each thread a few neighbours
  int most = 0;
  const int each = (pairs + kWarps * 32 - 1) / (kWarps * 32), my_first = min(pairs, tid * each), my_last = min(pairs, my_first + each);
  auto sum_before = [&](int sum) {  // of the threads before this one; a barrier stands between what was done ahead of the call and what comes after it
    int x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scratch[warp] = x;
    __syncthreads();
    int start = x - sum;
    for (int w = 0; w < warp; ++w) start += scratch[w];
    return start;
  };
  {
    int sum = 0;
    if (tid == 0) scratch[kWarps] = 0;
    for (int i = my_first; i < my_last; ++i) {
      Tile tile;
      open(tile, i, 0);
      int n = 0;
      if (tile.first_row < tile.rows) {
        const int key1 = tile.position(p, min(tile.first_row + kRows, tile.rows) - 1) + 1;
        if (key1 > 0) n = ((key1 + KV4_BLOCK - 1) / KV4_BLOCK - first_record(tile) + kRecords - 1) / kRecords;
      }
      shares.before[i] = sum;  // completed below
      sum += n;
      most = max(most, n);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const int start = sum_before(sum);
    if (lane == 0) atomicMax(&scratch[kWarps], most);
    for (int i = my_first; i < my_last; ++i) shares.before[i] += start;
    if (tid == kWarps * 32 - 1) shares.before[pairs] = start + sum;
    __syncthreads();
    most = scratch[kWarps];
  }
  // rows of pairs without any visible key: zeros
  for (int i = blockIdx.x; i < pairs; i += gridDim.x) {
    if (shares.before[i + 1] > shares.before[i]) continue;
    Tile tile;
    for (int head = 0; head < p.nkv; ++head) {
      open(tile, i, head);
      for (int x = tid; x < kRows * (D / 4); x += kWarps * 32) {
        const int row = tile.first_row + x / (D / 4);
        if (row < tile.rows) write_row<T>(p, tile, row, x % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f), kLowest, 0.f);
      }
    }
  }
  int total = shares.before[pairs] * p.nkv;
  // At least a step for every warp (of a short range no more than the range), no more parts of a range than pay (one CTA joins them, kRounds times eight
  // at once: a warp's step costs about as much as the joining of 20 / kRounds parts) and none over more than kMaxParts CTAs.
  constexpr int kRounds = (kRows * (D / 4) + kWarps * 32 - 1) / (kWarps * 32);
  const int least = max(max(min(kWarps, most), (int)sqrtf(0.2f * kRounds * most)), (most + kMaxParts - 1) / kMaxParts);
  int share = max(least, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  // Where it costs a warp no more than one step, a CTA has one range only: every range is counted as a whole number of shares.  (A second range in a
  // CTA costs its queries, its joining and two barriers: us without and with this rule, 32 query and 8 key heads, one request of 517 rows 11.4 / 8.8, of
  // 2,048 10.2 / 10.4, of 15,000 20.2 / 17.2; its last 4 tokens, 16 rows a key head: 1,900 24.5 / 17.1, 8,192 30 / 26; a prompt of 10 tokens 19.5 / 7.9.)
  const int spare = (int)gridDim.x - pairs * p.nkv;
  if (spare > 0 && total > 0) {
    const int whole = max(least, (total + spare - 1) / spare);
    if (whole <= share + kWarps) {
      share = whole;
      auto parts_of = [&](int n) { return (n + share - 1) / share; };
      if (total == most * pairs * p.nkv) {  // ranges of one length
        if (most % share != 0) {
          const int each_range = parts_of(most) * share;
          __syncthreads();
          for (int i = my_first; i < my_last; ++i) shares.before[i] = i * each_range;
          if (tid == kWarps * 32 - 1) shares.before[pairs] = pairs * each_range;
          __syncthreads();
        }
      } else {
        const int behind = shares.before[my_last];
        int sum = 0;
        for (int i = my_first; i < my_last; ++i) sum += parts_of((i + 1 < my_last ? shares.before[i + 1] : behind) - shares.before[i]) * share;
        int start = sum_before(sum), from = my_first < my_last ? shares.before[my_first] : 0;
        for (int i = my_first; i < my_last; ++i) {
          const int next = i + 1 < my_last ? shares.before[i + 1] : behind;
          shares.before[i] = start;
          start += parts_of(next - from) * share;
          from = next;
        }
        if (tid == kWarps * 32 - 1) shares.before[pairs] = start;
        __syncthreads();
      }
      total = shares.before[pairs] * p.nkv;
    }
  }
  const int begin = (int)min((long long)share * blockIdx.x, (long long)total), end = min(begin + share, total);
  if (begin >= end) return;
  auto pair_of = [&](int step) {
    int lo = 0, hi = pairs - 1;  // the last pair that begins at or before the step (pairs without keys begin with the next one)
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (shares.before[mid] * p.nkv <= step) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };

  // ---- a warp's steps: begin + warp, + kWarps, ...; lane i looks up where the i-th of its next 32 records lies, one round ahead
  constexpr uint32_t kNone = 0xffffffffu;
  auto look_up = [&](int record) -> uint32_t {  // counted over the warp's steps
    const int step = begin + warp + record / kRecords * kWarps;
    if (step >= end) return kNone;
    const int pair = pair_of(step), n = shares.before[pair + 1] - shares.before[pair], at = step - shares.before[pair] * p.nkv;
    const int head = at / n;
    Tile tile;
    open(tile, pair, head);
    const int blk = first_record(tile) + at % n * kRecords + record % kRecords;
    if (blk * KV4_BLOCK >= tile.context) return kNone;  // (an odd number of records)
    const int page = p.table[(size_t)(pair / p.row_tiles) * p.table_stride + blk / p.page_blocks];
    return ((uint32_t)min(max(page, 0), p.num_pages - 1) * p.nkv + head) * p.page_blocks + blk % p.page_blocks;
  };
  const int mine = begin + warp;
  uint32_t here = look_up(lane), ahead = look_up(32 + lane);
  uint8_t* ring = smem + warp * (kRing * Rec::kBytes);
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
  const uint8_t* pool_at = p.pool + lane * 16;
  constexpr int kStages = kRing / kRecords;
  int fetched = 0;  // records asked for
  auto fetch = [&]() {
#pragma unroll
    for (int r = 0; r < kRecords; ++r) {
      const uint32_t which = __shfl_sync(0xffffffffu, here, (fetched + r) & 31);
      if (which != kNone) {
        const uint8_t* src = pool_at + (size_t)which * Rec::kBytes;
        const uint32_t dst = ring_at + (fetched % kRing + r) * Rec::kBytes;
#pragma unroll
        for (int i = 0; i < Rec::kBytes / 512; ++i) copy16(dst + i * 512, src + i * 512);
        if (Rec::kBytes % 512 && lane < Rec::kBytes % 512 / 16) copy16(dst + Rec::kBytes / 512 * 512, src + Rec::kBytes / 512 * 512);
      }
    }
    copy_commit();
    fetched += kRecords;
    if ((fetched & 31) == 0) {
      here = ahead;
      ahead = look_up(fetched + 32 + lane);
    }
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  int done = 0;  // steps worked on
  for (int seg = begin; seg < end;) {
    const int pair = pair_of(seg), n_pair = shares.before[pair + 1] - shares.before[pair];
    const int head = (seg - shares.before[pair] * p.nkv) / n_pair, base = shares.before[pair] * p.nkv + head * n_pair;
    const int seg_end = min(end, base + n_pair);
    Tile tile;
    open(tile, pair, head);
    const int first_pos = tile.position(p, tile.first_row), last_pos = tile.position(p, min(tile.first_row + kRows, tile.rows) - 1);
    const int key0 = p.window > 0 ? max(0, first_pos - p.window + 1) : 0, blk0 = key0 / KV4_BLOCK;
    // keys that every row sees: [all0, all1)
    const int all0 = p.window > 0 ? last_pos - p.window + 1 : 0, all1 = first_pos + 1;

    // the queries as the products' second operand, one copy for all warps
    if (warp < kTiles) {
      uint32_t qf[kQ][D / 16][2];
      const int row = tile.first_row + 8 * warp + (kTwice ? g & 3 : g);
      kv4_query_row<D, kQ>(row < tile.rows ? tile.query<T>(p, row) + t * (D / 4) : nullptr, qf);
#pragma unroll
      for (int k = 0; k < kQ; ++k)
#pragma unroll
        for (int w = 0; w < D / 32; ++w)
          sq[((warp * kQ + k) * (D / 32) + w) * 32 + lane] = make_uint4(qf[k][2 * w][0], qf[k][2 * w][1], qf[k][2 * w + 1][0], qf[k][2 * w + 1][1]);
    }
    __syncthreads();
    float o[kTiles][D / 16][4], m[kTiles][2], l[kTiles][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      m[n][0] = m[n][1] = kLowest, l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    for (; mine + done * kWarps < seg_end; ++done) {
      fetch();
      copy_wait<kStages - 1>();
      __syncwarp();
      const uint8_t* rec = ring + (done % kStages) * (kRecords * Rec::kBytes);
      float s[kRecords][kTiles][4];
#pragma unroll
      for (int r = 0; r < kRecords; ++r)
        kv4_scores<D, kTiles, kQ>(rec + r * Rec::kBytes, rec + r * Rec::kBytes + Rec::kKeyScales,
                                  [&](int n, int part, int w) { return sq[((n * kQ + part) * (D / 32) + w) * 32 + lane]; }, s[r], g, t);
      const int key = (blk0 + (mine + done * kWarps - base) * kRecords) * KV4_BLOCK;
      const bool edge = key < all0 || key + kRecords * KV4_BLOCK > all1;
      bool grows = false;
      float top[kTiles][2];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
#pragma unroll
        for (int r = 0; r < kRecords; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[r][n][i] *= p.scale;
        if (edge) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int row = tile.first_row + 8 * n + (2 * t + c) % kColumnRows, pos = row < tile.rows ? tile.position(p, row) : -1;
#pragma unroll
            for (int r = 0; r < kRecords; ++r)
#pragma unroll
              for (int i = c; i < 4; i += 2) {
                const int at = key + r * KV4_BLOCK + g + 4 * (i - c);
                if (at > pos || (p.window > 0 && at <= pos - p.window)) s[r][n][i] = -INFINITY;
              }
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[n][c] = fmaxf(s[0][n][c], s[0][n][c + 2]);
#pragma unroll
          for (int r = 1; r < kRecords; ++r) top[n][c] = fmaxf(top[n][c], fmaxf(s[r][n][c], s[r][n][c + 2]));
          grows |= top[n][c] > m[n][c] + 8.f;
        }
      }
      // The maximum moves only when a score passes it by 2^8: until then weights up to 256 are as exact as those up to 1.
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = top[n][c];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            x = fmaxf(x, m[n][c]);
            const float f = kv4_exp2(m[n][c] - x);
            m[n][c] = x;
            l[n][c] *= f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[n][i][c] *= f, o[n][i][c + 2] *= f;
          }
      }
#pragma unroll
      for (int r = 0; r < kRecords; ++r) {
        uint32_t pf[kTiles][kParts][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = kv4_exp2(s[r][n][i] - m[n][i & 1]);
            l[n][i & 1] += w[i];
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t parts[kP];
            kv4_split<kP>(w[2 * i], w[2 * i + 1], parts);
            if constexpr (kTwice) {
              pf[n][0][i] = transpose8x8(t < 2 ? parts[0] : parts[1]);
            } else {
#pragma unroll
              for (int k = 0; k < kP; ++k) pf[n][k][i] = transpose8x8(parts[k]);
            }
          }
        }
        const int from = key + r * KV4_BLOCK;
        if (edge) add_values<kTiles, kParts, true>(rec + r * Rec::kBytes, pf, o, g, t, key0 - from, last_pos + 1 - from);
        else add_values<kTiles, kParts, false>(rec + r * Rec::kBytes, pf, o, g, t, 0, KV4_BLOCK);
      }
      __syncwarp();
    }

    // ---- the warps' parts of the segment meet in shared memory (behind the rings, which are being filled)
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[n][c];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int row = 8 * n + (2 * t + c) % kColumnRows;
        if (g == 0 && (!kTwice || t < 2)) sm[warp * kRows + row] = m[n][c], sl[warp * kRows + row] = x;
        float2* dst = reinterpret_cast<float2*>(so + (warp * kRows + row) * D + g * (D / 8));
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          float2 v = make_float2(o[n][i][c], o[n][i][c + 2]);
          if constexpr (kTwice) {  // both parts' sums, half of the lanes' pairs written by each of the two lanes that hold them
            v.x += __shfl_xor_sync(0xffffffffu, v.x, 2), v.y += __shfl_xor_sync(0xffffffffu, v.y, 2);
            if ((i & 1) == t >> 1) dst[i] = v;
          } else {
            dst[i] = v;
          }
        }
      }
    __syncthreads();
    const bool whole = seg == base && seg_end == base + n_pair;
    // (a CTA holds at most two ranges in part: the one it begins with, in its first place, and the one it ends with)
    float* part = p.part + ((size_t)blockIdx.x * 2 + (seg > begin ? 1 : 0)) * kRows * (D + 4);
    for (int i = tid; i < kRows * (D / 4); i += kWarps * 32) {
      const int r = i / (D / 4), channel = i % (D / 4) * 4, row = tile.first_row + r;
      if (row >= tile.rows) continue;
      RowSum sum;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum.m = fmaxf(sum.m, sm[w * kRows + r]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        sum.add(sm[w * kRows + r], sl[w * kRows + r], *reinterpret_cast<const float4*>(so + (w * kRows + r) * D + channel), sum.m);
      if (whole) {
        write_row<T>(p, tile, row, channel, sum.o, sum.m, sum.l);
      } else {
        *reinterpret_cast<float4*>(part + r * (D + 4) + 4 + channel) = sum.o;
        if (channel == 0) *reinterpret_cast<float2*>(part + r * (D + 4)) = make_float2(sum.m, sum.l);
      }
    }
    if (!whole) {
      // The CTA that comes last adds the range's parts up, in the order of the CTAs, and leaves its ticket at zero again.
      __syncthreads();
      const int c0 = base / share, c1 = (base + n_pair - 1) / share;
      if (tid == 0) {
        int* ticket = p.tickets + pair * p.nkv + head;
        int before;  // (release: the barrier puts the whole CTA's writes before it; acquire: the other CTAs' are seen behind the next barrier)
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
        const bool last = before == c1 - c0;
        if (last) *ticket = 0;
        scratch[kWarps + 1] = last;
      }
      __syncthreads();
      if (scratch[kWarps + 1]) {
        for (int i = tid; i < kRows * (D / 4); i += kWarps * 32) {
          const int r = i / (D / 4), channel = i % (D / 4) * 4, row = tile.first_row + r;
          if (row >= tile.rows) continue;
          const float* from = p.part + ((size_t)c0 * 2 * kRows + r) * (D + 4);
          const int skip = base > c0 * share ? kRows * (D + 4) : 0;  // the first CTA may have begun with another range
          constexpr int kStep = 2 * kRows * (D + 4), kAhead = 8;  // parts whose loads are in flight together
          RowSum sum;
          for (int first = 0; first <= c1 - c0; first += kAhead) {
            float2 ml[kAhead];
            float4 v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
              const int c = first + i;
              const float* x = from + (size_t)c * kStep + (c == 0 ? skip : 0);
              ml[i] = make_float2(kLowest, 0.f), v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (c <= c1 - c0) ml[i] = __ldcg(reinterpret_cast<const float2*>(x)), v[i] = __ldcg(reinterpret_cast<const float4*>(x + 4 + channel));
            }
            float top = sum.m;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) top = fmaxf(top, ml[i].x);
            RowSum next;
            next.m = top;
            next.add(sum.m, sum.l, sum.o, top);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) next.add(ml[i].x, ml[i].y, v[i], top);
            sum = next;
          }
          write_row<T>(p, tile, row, channel, sum.o, sum.m, sum.l);
        }
      }
    }
    __syncthreads();
    seg = seg_end;
  }
  copy_wait<0>();
}

// ---------------------------------------------------------------------------
// weights: w_j += sum over the rows r of exp(s_rj - lse_r).  A warp owns 16 keys of one head at a time.

// Few rows (kTiles tiles of 8): the warp goes over records kWarps * gridDim.x apart, the next one's codes on their way while it works on
// one; a key's sum is complete when its record is done, and is added without being read first (no other warp of the launch adds to it, unless requests
// share its page, so its value does not depend on any order).  Only the keys' half of a record is read, in words straight to registers: no shared memory, no barrier.
// Bound like attention_kernel by unpacking; 16 requests of up to 4,096 rows, 4 query rows a key head: 14 us (45 MB with the sums).
template <typename T, int kQ, int kTiles>
__global__ void __launch_bounds__(kWarps * 32) weights_kernel(const Params p, float* sums, int first_row) {
  ts_pdl_prologue();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  Tile tile;
  tile.open(p, blockIdx.z, blockIdx.y);
  if (first_row >= tile.rows || tile.context <= 0) return;
  const int rows = min(8 * kTiles, tile.rows - first_row), first_pos = tile.position(p, first_row), last_pos = tile.position(p, first_row + rows - 1);
  if (last_pos < 0) return;
  const int begin = p.window > 0 ? max(0, first_pos - p.window + 1) / KV4_BLOCK : 0, end = last_pos / KV4_BLOCK + 1;
  const int step = kWarps * gridDim.x, page_size = p.page_blocks * KV4_BLOCK;
  const int* table = p.table + (size_t)tile.b * p.table_stride;
  int blk = begin + blockIdx.x * kWarps + warp;
  if (blk >= end) return;

  constexpr int kWords = D / 32;
  struct Codes {
    uint32_t w[2][kWords], sc[2];
  };
  auto load = [&](int page, int at, Codes& c) {
    const uint8_t* rec = record(p, page, at, tile.head);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t* from = reinterpret_cast<const uint32_t*>(rec + (g + 8 * r) * (D / 2) + t * (D / 8));
      const uint8_t* scale = rec + Rec::kKeyScales + (g + 8 * r) * (D / 16) + t * (D / 64);
      if constexpr (kWords == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(from);
        c.w[r][0] = v.x, c.w[r][1] = v.y, c.sc[r] = *scale;
      } else {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(from + i);
          c.w[r][i] = v.x, c.w[r][i + 1] = v.y, c.w[r][i + 2] = v.z, c.w[r][i + 3] = v.w;
        }
        if constexpr (kWords == 4) c.sc[r] = *reinterpret_cast<const uint16_t*>(scale);
        else c.sc[r] = *reinterpret_cast<const uint32_t*>(scale);
      }
    }
  };
  int page = table[blk / p.page_blocks], next_page = blk + step < end ? table[(blk + step) / p.page_blocks] : 0;
  Codes codes;
  load(page, blk, codes);
  uint32_t qf[kTiles][kQ][D / 16][2];
  float lse[kTiles][2];
  int pos[kTiles][2];
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const int row = 8 * n + g;
    kv4_query_row<D, kQ>(row < rows ? tile.query<T>(p, first_row + row) + t * (D / 4) : nullptr, qf[n]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = 8 * n + 2 * t + c;
      lse[n][c] = INFINITY, pos[n][c] = -1;  // a row that does not exist gives no weight
      if (r < rows) {
        lse[n][c] = p.lse[(size_t)tile.token(p, first_row + r) * p.nq + tile.query_head(p, first_row + r)] * kLog2e;
        pos[n][c] = tile.position(p, first_row + r);
      }
    }
  }
  const int all0 = p.window > 0 ? last_pos - p.window + 1 : 0, all1 = first_pos + 1;  // keys that every row sees
  while (true) {
    Codes next;
    const int next_blk = blk + step;
    if (next_blk < end) load(next_page, next_blk, next);
    const int page_after = next_blk + step < end ? table[(next_blk + step) / p.page_blocks] : 0;
    float s[kTiles][4];
    kv4_scores_of<D, kTiles, kQ>(
        codes.w, codes.sc,
        [&](int n, int part, int i) { return make_uint4(qf[n][part][2 * i][0], qf[n][part][2 * i][1], qf[n][part][2 * i + 1][0], qf[n][part][2 * i + 1][1]); }, s);
    const int key = blk * KV4_BLOCK;
    float w[2] = {0.f, 0.f};
    const bool edge = rows < 8 * kTiles || key < all0 || key + KV4_BLOCK > all1;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = i & 1, at = key + g + 8 * (i >> 1);
        const float e = kv4_exp2(fmaf(s[n][i], p.scale, -lse[n][c]));
        if (!edge || (at <= pos[n][c] && (p.window == 0 || at > pos[n][c] - p.window))) w[i >> 1] += e;
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] += __shfl_xor_sync(0xffffffffu, w[i], 1);
      w[i] += __shfl_xor_sync(0xffffffffu, w[i], 2);
    }
    const int at = key + g + 8 * (t & 1);
    if (t < 2 && at < tile.context)
      atomicAdd(sums + ((size_t)min(max(page, 0), p.num_pages - 1) * p.nkv + tile.head) * page_size + at % page_size, t == 0 ? w[0] : w[1]);
    if (next_blk >= end) break;
    blk = next_blk, page = next_page, next_page = page_after, codes = next;
  }
}

// The same for many rows (portions of prompts).  A CTA owns 128 keys (64 for heads of 256): its warps keep their keys
// unpacked in registers, kKeyWarps of them side by side, while the query rows pass through shared memory, 64 at a time and
// twice buffered; kRowWarps warps share a key and take the rows in turns, and add up at the end in one order.
constexpr int kKeyTiles = D <= 128 ? 2 : 1;  // of 16 keys per warp
constexpr int kKeyWarps = 4, kRowWarps = 4, kStageRows = 64;
constexpr int kChunkKeys = kKeyWarps * kKeyTiles * 16, kWeightThreads = kKeyWarps * kRowWarps * 32;

template <int kQ>
struct WeightsStage {
  static constexpr int kBytes = kQ * kStageRows * D * 2 + kStageRows * 8;
};

template <typename T, int kQ>
__global__ void __launch_bounds__(kWeightThreads, 1) weights_rows_kernel(const Params p, float* sums) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float meet[kRowWarps][kChunkKeys];
  constexpr int kStage = WeightsStage<kQ>::kBytes, kChunks = D / 8;  // 16-byte pieces of a row
  ts_pdl_prologue();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int key_warp = warp % kKeyWarps, row_warp = warp / kKeyWarps;
  Tile tile;
  tile.open(p, blockIdx.z, blockIdx.y);
  const int chunk_key = blockIdx.x * kChunkKeys, before = tile.context - tile.q_len;
  if (chunk_key >= tile.context) return;
  const int last_key = min(chunk_key + kChunkKeys, tile.context) - 1;
  const int first_token = max(0, chunk_key - before);
  const int tokens = p.window > 0 ? min(tile.q_len, last_key + p.window - before) : tile.q_len;
  if (first_token >= tokens) return;
  const int first_row = first_token * p.group, rows = tokens * p.group;

  // this warp's keys: word u = 4w + t of a row holds the channels 8u..8u+7, unpacked as the pairs (0,1) (2,3) (4,5) (6,7)
  const int key = chunk_key + key_warp * kKeyTiles * 16;
  uint32_t a[kKeyTiles][D / 32][2][4];
#pragma unroll
  for (int m = 0; m < kKeyTiles; ++m) {
    const int blk = key / KV4_BLOCK + m;
    const bool there = blk * KV4_BLOCK < tile.context;
    const uint8_t* rec = record(p, there ? p.table[(size_t)tile.b * p.table_stride + blk / p.page_blocks] : 0, blk, tile.head);
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const int u = 4 * w + t;
        const uint32_t x = *reinterpret_cast<const uint32_t*>(rec + (g + 8 * r) * (D / 2) + 4 * u);
        const uint32_t sc = rec[Rec::kKeyScales + (g + 8 * r) * (D / 16) + u / 2];
        __nv_bfloat162 f, c;
        kv4_factors(sc, sc, f, c);
        const uint32_t p0 = kv4_pair(x << 3, f, c), p1 = kv4_pair(x >> 1, f, c), p2 = kv4_pair(x >> 5, f, c), p3 = kv4_pair(x >> 9, f, c);
        a[m][w][r][0] = __byte_perm(p0, p1, 0x5410), a[m][w][r][1] = __byte_perm(p2, p3, 0x5410);
        a[m][w][r][2] = __byte_perm(p0, p1, 0x7632), a[m][w][r][3] = __byte_perm(p2, p3, 0x7632);
      }
  }

  // A stage: its rows [part][64][D] bfloat16, the 16-byte piece c of row r at c ^ (r & 1) * 4 (eight lanes of a warp's read
  // then fall on eight different groups of banks), then every row's logarithm and last visible key.
  const uint32_t smem_at = (uint32_t)__cvta_generic_to_shared(smem);
  auto fetch = [&](int stage, int base) {
    uint8_t* buf = smem + stage * kStage;
    for (int i = threadIdx.x; i < kStageRows * kChunks; i += kWeightThreads) {
      const int r = i / kChunks, c = i % kChunks, at = r * D * 2 + ((c ^ ((r & 1) * 4)) * 16);
      const bool there = base + r < rows;
      const T* src = tile.query<T>(p, there ? base + r : first_row) + c * 8;
      if constexpr (sizeof(T) == 2) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_at + stage * kStage + at), "l"(src), "r"(there ? 16 : 0));
      } else {
        const float4 lo = reinterpret_cast<const float4*>(src)[0], hi = reinterpret_cast<const float4*>(src)[1];
        const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        uint32_t parts[4][kQ];
#pragma unroll
        for (int j = 0; j < 4; ++j) kv4_split<kQ>(there ? x[2 * j] : 0.f, there ? x[2 * j + 1] : 0.f, parts[j]);
#pragma unroll
        for (int k = 0; k < kQ; ++k)
          *reinterpret_cast<uint4*>(buf + k * kStageRows * D * 2 + at) = make_uint4(parts[0][k], parts[1][k], parts[2][k], parts[3][k]);
      }
    }
    if (threadIdx.x < kStageRows) {
      const int row = base + threadIdx.x;
      float lse = INFINITY;  // a row that does not exist gives no weight
      int pos = -1;
      if (row < rows) lse = p.lse[(size_t)tile.token(p, row) * p.nq + tile.query_head(p, row)] * kLog2e, pos = tile.position(p, row);
      reinterpret_cast<float2*>(buf + kQ * kStageRows * D * 2)[threadIdx.x] = make_float2(lse, __int_as_float(pos));
    }
    copy_commit();
  };

  float w[kKeyTiles][2];
#pragma unroll
  for (int m = 0; m < kKeyTiles; ++m) w[m][0] = w[m][1] = 0.f;
  fetch(0, first_row);
  int stage = 0;
  for (int base = first_row; base < rows; base += kStageRows, stage ^= 1) {
    if (base + kStageRows < rows) fetch(stage ^ 1, base + kStageRows);
    else copy_commit();
    copy_wait<1>();
    __syncthreads();
    const uint8_t* buf = smem + stage * kStage;
    const float2* info = reinterpret_cast<const float2*>(buf + kQ * kStageRows * D * 2);
#pragma unroll 1
    for (int n = row_warp * 8; n < kStageRows && base + n < rows; n += kRowWarps * 8) {
      float s[kKeyTiles][4];
#pragma unroll
      for (int m = 0; m < kKeyTiles; ++m) s[m][0] = s[m][1] = s[m][2] = s[m][3] = 0.f;
#pragma unroll
      for (int k = 0; k < kQ; ++k)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint4 q = *reinterpret_cast<const uint4*>(buf + k * kStageRows * D * 2 + (n + g) * D * 2 + (((4 * i + t) ^ ((g & 1) * 4)) * 16));
#pragma unroll
          for (int m = 0; m < kKeyTiles; ++m) kv4_mma(s[m], a[m][i][0][0], a[m][i][1][0], a[m][i][0][1], a[m][i][1][1], q.x, q.y);
#pragma unroll
          for (int m = 0; m < kKeyTiles; ++m) kv4_mma(s[m], a[m][i][0][2], a[m][i][1][2], a[m][i][0][3], a[m][i][1][3], q.z, q.w);
        }
      const float2 r0 = info[n + 2 * t], r1 = info[n + 2 * t + 1];
      const int p0 = __float_as_int(r0.y), p1 = __float_as_int(r1.y);
      // (positions grow with the rows)
      const int low = __float_as_int(info[n].y), high = __float_as_int(info[min(n + 7, rows - 1 - base)].y);
      const bool all = low >= key + kKeyTiles * 16 - 1 && (p.window == 0 || high - p.window < key);
#pragma unroll
      for (int m = 0; m < kKeyTiles; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = key + 16 * m + g + 8 * i;
          const float e0 = kv4_exp2(fmaf(s[m][2 * i], p.scale, -r0.x)), e1 = kv4_exp2(fmaf(s[m][2 * i + 1], p.scale, -r1.x));
          if (all) {
            w[m][i] += e0 + e1;
          } else {
            if (at <= p0 && (p.window == 0 || at > p0 - p.window)) w[m][i] += e0;
            if (at <= p1 && (p.window == 0 || at > p1 - p.window)) w[m][i] += e1;
          }
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int m = 0; m < kKeyTiles; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[m][i] += __shfl_xor_sync(0xffffffffu, w[m][i], 1);
      w[m][i] += __shfl_xor_sync(0xffffffffu, w[m][i], 2);
      if (t == 0) meet[row_warp][(key_warp * kKeyTiles + m) * 16 + g + 8 * i] = w[m][i];
    }
  __syncthreads();
  const int at = chunk_key + threadIdx.x;
  if (threadIdx.x < kChunkKeys && at < tile.context) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kRowWarps; ++i) sum += meet[i][threadIdx.x];
    const int page_size = p.page_blocks * KV4_BLOCK, page = p.table[(size_t)tile.b * p.table_stride + at / page_size];
    // (A key that nobody sees is left alone: its page may have been given back.  One add to a key of a page that requests do not share, so in one order.)
    if (sum != 0.f) atomicAdd(sums + ((size_t)min(max(page, 0), p.num_pages - 1) * p.nkv + tile.head) * page_size + at % page_size, sum);
  }
}

template <typename T, int kQ>
int launch_weights(const Params& p, float* sums, int num_seqs, int max_context, int max_q, cudaStream_t stream) {
  // Streamed: a record is read, used and done with, by as many warps as run at once, for kPass rows at a time (their registers hold so many queries).
  // Else keys are unpacked once, 128 of a head to a CTA, which pays where those CTAs are few or the rows many.  us streamed / unpacked once, 16 requests
  // of 4,096 rows, 24 / 64 / 128 query rows: bfloat16 heads of 64 35 / 117, 64 / 130, 122 / 166, of 256 79 / 281, 174 / 315, 343 / 420; float32 of
  // 128 79 / 156, 180 / 199, 355 / 299; one request of 2,048 rows, bfloat16 heads of 128: 10 / 10, 17 / 12, 33 / 14.  (Of bfloat16 heads of 128 only
  // up to 48 rows come here: ops.py.)
  constexpr int kPass = kQ == 1 && D <= 128 ? 32 : 16, kStreamed = kQ == 1 ? 128 : 64;
  const int rows = max_q * p.group, passes = (rows + kPass - 1) / kPass;
  if (passes == 1 || (rows <= kStreamed && (long long)((max_context + 127) / 128) * p.nkv * num_seqs > 148 * passes)) {
    const int most = (max_context + KV4_BLOCK * kWarps - 1) / (KV4_BLOCK * kWarps), want = 8 * 148 / (p.nkv * num_seqs) + 1;
    const dim3 grid(most < want ? most : want, p.nkv, num_seqs);
    for (int first = 0; first < rows; first += kPass) {
      int status;
      if (rows - first <= 8) status = ts_launch(weights_kernel<T, kQ, 1>, grid, dim3(kWarps * 32), 0, stream, p, sums, first);
      else if (kPass == 16 || rows - first <= 16) status = ts_launch(weights_kernel<T, kQ, 2>, grid, dim3(kWarps * 32), 0, stream, p, sums, first);
      else status = ts_launch(weights_kernel<T, kQ, kPass / 8>, grid, dim3(kWarps * 32), 0, stream, p, sums, first);
      if (status) return status;
    }
    return 0;
  }
  constexpr int smem = 2 * WeightsStage<kQ>::kBytes;
  static bool set = false;
  if (!set) {
    cudaError_t e = cudaFuncSetAttribute(weights_rows_kernel<T, kQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    set = true;
  }
  const dim3 grid((max_context + kChunkKeys - 1) / kChunkKeys, p.nkv, num_seqs);
  return ts_launch(weights_rows_kernel<T, kQ>, grid, dim3(kWeightThreads), smem, stream, p, sums);
}

template <typename T, int kTiles, int kQ, int kP, int kRecords, bool kTwice = false>
struct Attention {
  static constexpr int kRows = kTwice ? 4 : 8 * kTiles;
  static constexpr int kSmem = kWarps * kRing * Rec::kBytes + kTiles * kQ * D * 16 + kWarps * kRows * (D + 2) * 4;  // and 4 bytes per pair
  static constexpr int kFewPairs = 256;
  // CTAs that run at once on the device (with at most kFewPairs pairs), or a negative error
  static int ctas() {
    static int n = 0;
    if (n == 0) {
      int device = 0, sms = 0, per_sm = 0;
      cudaError_t e = cudaFuncSetAttribute(attention_kernel<T, kTiles, kQ, kP, kRecords, kTwice>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           kSmem + (kMaxTiles + 1) * 4);
      if (e == cudaSuccess) e = cudaGetDevice(&device);
      if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
      if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attention_kernel<T, kTiles, kQ, kP, kRecords, kTwice>, kWarps * 32,
                                                                                kSmem + (kFewPairs + 1) * 4);
      if (e != cudaSuccess) return -(int)e - 100;
      n = sms * (per_sm > 0 ? per_sm : 1);
    }
    return n;
  }
  static int launch(const Params& p, int grid, cudaStream_t stream) {
    return ts_launch(attention_kernel<T, kTiles, kQ, kP, kRecords, kTwice>, dim3(grid), dim3(kWarps * 32), kSmem + (p.num_seqs * p.row_tiles + 1) * 4, stream, p);
  }
};

}  // namespace

using AttentionFloat = Attention<float, 1, 3, 3, 1>;
using AttentionFew = Attention<__nv_bfloat16, 1, 1, 2, D <= 128 ? 2 : 1>;
using AttentionFour = Attention<__nv_bfloat16, 1, 1, 2, D <= 128 ? 2 : 1, true>;
#if TS_HEAD_DIM <= 128
using AttentionMore = Attention<__nv_bfloat16, 2, 1, 2, 1>;
#endif

// How many rows a tile has, by the type and the rows of a sequence and key head.
static int tile_rows(int dtype, int rows) { return dtype != TS_DTYPE_BF16 ? 8 : rows <= 4 ? 4 : rows > 8 && D <= 128 ? 16 : 8; }

// CTAs of a launch (at most), for the size of `part`: grid * 2 * tile rows * (D + 4) floats; negative: an error.
static int grid_of(int dtype, int rows) {
  if (dtype == TS_DTYPE_F32) return AttentionFloat::ctas();
  if (tile_rows(dtype, rows) == 4) return AttentionFour::ctas();
#if TS_HEAD_DIM <= 128
  if (tile_rows(dtype, rows) == 16) return AttentionMore::ctas();
#endif
  return AttentionFew::ctas();
}
TS_EXPORT long long ts_attention_kv4_part_floats(int dtype, int rows) {
  const int grid = grid_of(dtype, rows);
  return grid < 0 ? grid : (long long)grid * 2 * tile_rows(dtype, rows) * (D + 4);
}

// q, out [tokens][nq][D] of `dtype`, lse [tokens][nq] or null, sinks [nq] or null; part: see above; tickets: `num_tickets` zeros (zeros again
// afterwards).  Batches of more pairs than a launch or the tickets hold take several launches.
struct Kv4AttentionArgs {
  const void *q, *pool;
  void* out;
  float* lse;
  const float* sinks;
  const int *cu, *context, *table;
  float* part;
  int* tickets;
  void* stream;
  int dtype, table_stride, page_blocks, num_pages, tokens, num_seqs, max_q, nq, nkv, window, num_tickets;
  float scale;
};
TS_EXPORT int ts_attention_kv4(const Kv4AttentionArgs* args) {
  const auto [q, pool, out, lse, sinks, cu, context, table, part, tickets, stream, dtype, table_stride, page_blocks, num_pages, tokens, num_seqs, max_q, nq,
              nkv, window, num_tickets, scale] = *args;
  if (tokens < 1 || num_seqs < 1 || max_q < 1) return 0;
  if (num_tickets < nkv || (long long)max_q * (nq / nkv) > 0x7fffffffLL - 16) return TS_ERR_UNSUPPORTED_SIZE;
  const int rows = max_q * (nq / nkv), grid = grid_of(dtype, rows), row_tiles = (rows + tile_rows(dtype, rows) - 1) / tile_rows(dtype, rows);
  if (grid < 1) return -grid - 100;
  // pairs of a launch: their key ranges, counted in records over all heads, stay below 2^31
  const long long records = (long long)table_stride * page_blocks * nkv;
  long long most = kMaxTiles;
  if (most > num_tickets / nkv) most = num_tickets / nkv;
  if (most > 0x7fff0000LL / records) most = 0x7fff0000LL / records;
  if (most < 1) return TS_ERR_UNSUPPORTED_SIZE;
  const int tiles = (int)(most < row_tiles ? most : row_tiles), seqs = (int)(most / tiles);
  for (int b = 0; b < num_seqs; b += seqs)
    for (int tile = 0; tile < row_tiles; tile += tiles) {
      Params p = {q, (const uint8_t*)pool, out, lse, sinks, cu + b, context + b, table + (size_t)b * table_stride, part, tickets, table_stride, page_blocks,
                  num_pages, tokens, num_seqs - b < seqs ? num_seqs - b : seqs, nq, nkv, nq / nkv, window,
                  row_tiles - tile < tiles ? row_tiles - tile : tiles, tile, scale * kLog2e};
      int status;
      if (dtype == TS_DTYPE_F32) status = AttentionFloat::launch(p, grid, (cudaStream_t)stream);
      else if (tile_rows(dtype, rows) == 4) status = AttentionFour::launch(p, grid, (cudaStream_t)stream);
#if TS_HEAD_DIM <= 128
      else if (tile_rows(dtype, rows) == 16) status = AttentionMore::launch(p, grid, (cudaStream_t)stream);
#endif
      else status = AttentionFew::launch(p, grid, (cudaStream_t)stream);
      if (status) return status;
    }
  return 0;
}

struct Kv4WeightsArgs {
  const void *q, *pool;
  float *lse, *sums;
  const int *cu, *context, *table;
  void* stream;
  int dtype, table_stride, page_blocks, num_pages, tokens, num_seqs, max_q, max_context, nq, nkv, window;
  float scale;
};
TS_EXPORT int ts_attention_kv4_weights(const Kv4WeightsArgs* args) {
  const auto [q, pool, lse, sums, cu, context, table, stream, dtype, table_stride, page_blocks, num_pages, tokens, num_seqs, max_q, max_context, nq, nkv,
              window, scale] = *args;
  if (tokens < 1 || num_seqs < 1 || max_context < 1) return 0;
  if (num_seqs > 65535 || nkv > 65535) return TS_ERR_UNSUPPORTED_SIZE;
  Params p = {q, (const uint8_t*)pool, nullptr, lse, nullptr, cu, context, table, nullptr, nullptr, table_stride, page_blocks, num_pages, tokens, num_seqs, nq, nkv,
              nq / nkv, window, 1, 0, scale * kLog2e};
  if (dtype == TS_DTYPE_F32) return launch_weights<float, 3>(p, sums, num_seqs, max_context, max_q, (cudaStream_t)stream);
  return launch_weights<__nv_bfloat16, 1>(p, sums, num_seqs, max_context, max_q, (cudaStream_t)stream);
}
