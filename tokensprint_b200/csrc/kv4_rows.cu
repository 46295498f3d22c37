// Rows into the 4-bit cache, rows out of it, and the rows that stay when a request is cut to a budget.
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace {

// amax / 7 rounded to the scales a byte holds, as that byte (the nearest, ties to even; see kv4.cuh).
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const float t = amax / 7.f;
  if (!(t < 8192.f)) return 0xE0u;  // 8192 = 2^13: exponent 28
  const uint32_t u = __float_as_uint(t);
  if (t < 6.103515625e-05f) return (uint32_t)__float2int_rn(t * 131072.f);  // below 2^-14 in steps of 2^-17 (2^-14 itself: byte 8)
  const uint32_t r = u + 0x7ffffu + ((u >> 20) & 1u);  // to three bits of mantissa, a carry moves the exponent
  return (r >> 20) - ((127u - 15u) << 3);
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __half2float(__ushort_as_half((unsigned short)(byte << 7))); }

template <typename T>
__device__ __forceinline__ void read_group(const T* p, float (&x)[16]);
template <>
__device__ __forceinline__ void read_group<float>(const float* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = reinterpret_cast<const float4*>(p)[i];
    x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
  }
}
template <>
__device__ __forceinline__ void read_group<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 v = reinterpret_cast<const uint4*>(p)[i];
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) x[8 * i + 2 * j] = __uint_as_float(u[j] << 16), x[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
  }
}

// 16 values to codes (returned in w) and their scale's byte.
__device__ __forceinline__ uint32_t quantise(const float (&x)[16], uint2& w) {
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) asm("max.NaN.f32 %0, %0, %1;" : "+f"(amax) : "f"(fabsf(x[j])));
  uint32_t half[2] = {0u, 0u};
  const float t = amax / 7.f;
  if (t >= 6.103515625e-05f && t < 8192.f) {
    // A normal scale: |x / s| stays below 7.5.  The quotient is rounded as a division would, by Markstein's correction: with inv = 1/s rounded, q = x inv, then
    // q + (x - q s) inv, whose remainder is exact.  Adding 1.5 * 2^23 + 8 rounds it to a whole number, ties to even, and leaves the code in the low bits.
    const uint32_t byte = scale_byte(amax);
    const float s = scale_of(byte), inv = 1.f / s;
#pragma unroll
    for (int j = 15; j >= 0; --j) {
      float q = x[j] * inv;
      q = fmaf(fmaf(-q, s, x[j]), inv, q);
      half[j / 8] = (half[j / 8] << 4) | (__float_as_uint(q + 12582920.f) & 15u);
    }
    w = make_uint2(half[0], half[1]);
    return byte;
  }
  // NaN, infinities, the smallest and the largest scales
  float y[16];
  amax = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    y[j] = x[j] == x[j] ? x[j] : 0.f;
    amax = fmaxf(amax, fabsf(y[j]));
  }
  const uint32_t byte = scale_byte(amax);
  const float s = byte ? scale_of(byte) : 1.f;  // (a scale of zero: the whole group rounds to zero)
#pragma unroll
  for (int j = 15; j >= 0; --j) half[j / 8] = (half[j / 8] << 4) | (byte ? (uint32_t)(__float2int_rn(fminf(fmaxf(y[j] / s, -7.f), 7.f)) + 8) : 8u);
  w = make_uint2(half[0], half[1]);
  return byte;
}

// A thread takes the 16 channels of one group at a time: their largest, s = amax / 7 rounded, the codes 8 + x / s rounded, 8 + 1 bytes out; `width`
// threads (32 or 128) go over the groups of a token, keys first.  One pass, bound by memory: 2 bytes in and 9/16 out per value.  With many tokens
// it is the number of warps that hides the loads (16,384 tokens of 8 heads of 128: 21.7 us with a group at a time and 46 registers, 38.6 with
// four in flight and 125; 105 MB).  8,192 tokens: 15.4 us from cold caches, 2.8 TB/s; 8 tokens: 2.4 us, a launch and two trips to memory.
template <typename T>
__global__ void __launch_bounds__(128, 10) store_kernel(const T* k, const T* v, long long k_stride, long long v_stride, uint8_t* pool, float* sums,
                                                    const int* slots, int tokens, int nkv, int log_groups, int page_blocks, int num_slots, int width) {
  ts_pdl_prologue();
  const int groups = 1 << log_groups, d = 16 * groups, units = nkv << log_groups;
  const int token = blockIdx.x * (128 / width) + threadIdx.x / width;
  if (token >= tokens) return;
  const int slot = slots[token];
  if (slot < 0 || slot >= num_slots) return;
  const int page_size = page_blocks * KV4_BLOCK, page = slot / page_size, in_page = slot % page_size, row = in_page % KV4_BLOCK;
  uint8_t* records = pool + ((size_t)page * nkv * page_blocks + in_page / KV4_BLOCK) * (18 * d);  // head 0's
  const T *from_k = k + token * k_stride, *from_v = v + token * v_stride;
  for (int i = threadIdx.x % width; i < 2 * units; i += width) {
    float x[16];
    read_group<T>(i < units ? from_k + i * 16 : from_v + (i - units) * 16, x);
    const int unit = i < units ? i : i - units, head = unit >> log_groups, grp = unit & (groups - 1);
    uint2 w;
    const uint32_t byte = quantise(x, w);
    uint8_t* rec = records + (size_t)head * page_blocks * (18 * d) + (i < units ? 0 : 9 * d);
    *reinterpret_cast<uint2*>(rec + row * (d / 2) + grp * 8) = w;
    rec[8 * d + row * groups + grp] = (uint8_t)byte;
    if (sums != nullptr && i < units && grp == 0) sums[((size_t)page * nkv + head) * page_size + in_page] = 0.f;  // it has gathered no weight
  }
}

// A thread takes eight channels: 4 + 1 bytes in, one store of 16 bytes of bfloat16 out, a warp's stores one behind the other.  Bound by what
// it writes: 65,536 rows of 8 heads of 128 (268 MB out) take 58 us, 5.9 TB/s with the codes; 8,192 take 18 us.
template <typename T>
__global__ void __launch_bounds__(128) load_kernel(const uint8_t* pool, const int* slots, T* k, T* v, int rows, int nkv, int log_groups, int page_blocks,
                                                   int num_slots, int width) {
  ts_pdl_prologue();
  const int log_words = log_groups + 1, d = 8 << log_words, units = nkv << log_words;  // units of 8 channels
  const int row = blockIdx.x * (128 / width) + threadIdx.x / width;
  if (row >= rows) return;
  const int slot = slots[row];
  const bool there = slot >= 0 && slot < num_slots;
  const int page_size = page_blocks * KV4_BLOCK, page = there ? slot / page_size : 0, in_page = there ? slot % page_size : 0, at = in_page % KV4_BLOCK;
  const uint8_t* records = pool + ((size_t)page * nkv * page_blocks + in_page / KV4_BLOCK) * (18 * d);
  T *to_k = k + (size_t)row * units * 8, *to_v = v + (size_t)row * units * 8;
  constexpr int kAhead = 8;
  for (int first = threadIdx.x % width; first < 2 * units; first += kAhead * width) {
    uint32_t code[kAhead], scale[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int i = first + a * width, unit = i < units ? i : i - units, word = unit & ((1 << log_words) - 1);
      code[a] = scale[a] = 0u;
      if (there && i < 2 * units) {
        const uint8_t* rec = records + (size_t)(unit >> log_words) * page_blocks * (18 * d) + (i < units ? 0 : 9 * d);
        code[a] = *reinterpret_cast<const uint32_t*>(rec + at * (d / 2) + word * 4);
        scale[a] = rec[8 * d + at * (d / 16) + word / 2];
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int i = first + a * width;
      if (i >= 2 * units) break;
      T* dst = i < units ? to_k + i * 8 : to_v + (i - units) * 8;
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(dst) = kv4_unpack(code[a], scale[a]);
      } else {
        const float s = scale_of(scale[a]);
        const uint32_t c = code[a];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          reinterpret_cast<float4*>(dst)[j] = make_float4((float)((int)(c >> (16 * j) & 15u) - 8) * s, (float)((int)(c >> (16 * j + 4) & 15u) - 8) * s,
                                                          (float)((int)(c >> (16 * j + 8) & 15u) - 8) * s, (float)((int)(c >> (16 * j + 12) & 15u) - 8) * s);
      }
    }
  }
}

// The rows that a batch's queries can see, of heads of 128, as bfloat16 pages of 128 rows for the prompt attention, and the block table of those
// pages: request b has the pages [b * blocks, (b + 1) * blocks); out_lens: its rows, as many as have a place.  A CTA unpacks 64 rows of one head.
// Of a page that holds a visible key every row up to the request's last is written; the attention itself clears what lies behind that one.
// 2,048 rows of 8 heads: 6 us (2.4 MB in, 8.4 MB out), most of it the start and two trips to memory; the attention that follows reads them from the L2.
constexpr int kExpandRows = 64, kExpandPage = 128, kExpandDim = 128;
__global__ void __launch_bounds__(256) expand_kernel(const uint8_t* pool, const int* table, int table_stride, const int* cu, const int* context, uint4* k,
                                                     uint4* v, int* out_table, int* out_lens, uint4* out, float* lse, const float* sinks, int group, int nkv,
                                                     int page_blocks, int num_pages, int blocks, int window) {
  ts_pdl_prologue();
  constexpr int kWords = kExpandDim / 8, kUnits = kExpandRows * kWords * 2 / 256;
  const int b = blockIdx.z, head = blockIdx.y, first = blockIdx.x * kExpandRows;
  const int n = min(context[b], min(table_stride * page_blocks * KV4_BLOCK, blocks * kExpandPage));
  if (head == 0 && threadIdx.x == 0) {
    if (first % kExpandPage == 0) out_table[b * blocks + first / kExpandPage] = b * blocks + first / kExpandPage;
    if (first == 0) out_lens[b] = n;
  }
  const int queries = cu[b + 1] - cu[b], oldest = window > 0 ? n - queries - window + 1 : 0;  // the first key that some query sees
  // Tokens ahead of the first row see nothing: zeros, and the logarithm of nothing or of the sink.  The attention leaves out tiles that have no others.
  const int unseen = (queries - max(n, 0)) * group;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < unseen * kWords; i += gridDim.x * blockDim.x) {
    const int row = i / kWords, query_head = head * group + row % group;
    const size_t at = (size_t)(cu[b] + row / group) * (nkv * group) + query_head;
    out[at * kWords + i % kWords] = make_uint4(0u, 0u, 0u, 0u);
    if (lse != nullptr && i % kWords == 0) lse[at] = sinks != nullptr ? sinks[query_head] : -INFINITY;
  }
  // (The attention walks whole pages, from the first that holds a visible key on: what it reads ahead of that key weighs nothing, but has to be
  // numbers.  So only whole pages are left out.)
  const int page_end = first / kExpandPage * kExpandPage + kExpandPage;
  if (first >= n || page_end <= oldest || queries <= 0) return;
  uint32_t code[kUnits], scale[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int unit = threadIdx.x + 256 * i, word = unit % kWords, values = unit / (kExpandRows * kWords);
    const int row = min(first + unit / kWords % kExpandRows, n - 1), blk = row / KV4_BLOCK;
    const int page = min(max(table[(size_t)b * table_stride + blk / page_blocks], 0), num_pages - 1);
    const uint8_t* rec = pool + (((size_t)page * nkv + head) * page_blocks + blk % page_blocks) * (18 * kExpandDim) + values * 9 * kExpandDim;
    code[i] = *reinterpret_cast<const uint32_t*>(rec + row % KV4_BLOCK * (kExpandDim / 2) + word * 4);
    scale[i] = rec[8 * kExpandDim + row % KV4_BLOCK * (kExpandDim / 16) + word / 2];
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int unit = threadIdx.x + 256 * i, word = unit % kWords, values = unit / (kExpandRows * kWords);
    const int row = first + unit / kWords % kExpandRows;
    if (row < n) (values ? v : k)[(((size_t)b * blocks * kExpandPage + row) * nkv + head) * kWords + word] = kv4_unpack(code[i], scale[i]);
  }
}

// ---------------------------------------------------------------------------
// eviction

constexpr int kEvictThreads = 512, kEvictWarps = kEvictThreads / 32;
constexpr int kDigits = 2048;          // bins of a pass of the radix select: 11, 11 and 10 bits
constexpr int kKeptKeys = 16384;       // most weights kept in shared memory; of longer requests they are read again for every pass
constexpr int kMoveRows = 256;         // rows that a CTA moves at a time

// A weight as an unsigned number of the same order; NaN is the largest, both zeros are one.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The sum of `v` over the threads before this one; `total`: over all of them.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* scratch, uint32_t& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kEvictWarps; ++i) {
    const uint32_t s = scratch[i];
    if (i < warp) before += s;
    all += s;
  }
  __syncthreads();
  total = all;
  return before + x - v;
}

__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// Four words at `p` of this CTA's shared memory, as the CTA `rank` of the cluster has them.
__device__ __forceinline__ uint4 peer_words(const uint32_t* p, int rank) {
  uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
  uint4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// A cluster of CTAs per request and head, every CTA with an equal run of its rows.  The weights between the first and the recent rows are ranked by
// a radix select whose counts the CTAs add up from one another's shared memory; every kept row gets its new place, and its source is written
// down there.  Then the kept rows move forward in rounds, kMoveRows places per CTA: all reads of a round, a barrier of the cluster, its writes.
// That is safe in place: a row never moves backwards and the order is kept, so what a round writes lies before everything that later
// rounds read.  (Every CTA ranking all rows by itself took 35 us of 72 for 128 pairs of 8,190 rows.)  16 requests of up to 8,190 rows of 8 heads of 128 cut
// to 4,096: 41 us, where the rows that move (151 MB there and back) would take 23 at the copy rate; the rest is the ranking (three passes over
// weights in shared memory, each with barriers of the cluster) and rounds that wait for their own reads.  One request: 12 us, all of it such waits.
template <int D>
__global__ void __launch_bounds__(kEvictThreads, 3) evict_kernel(uint8_t* pool, float* sums, const int* table, int table_stride, const int* context,
                                                                 int* new_lens, int* order, int nkv, int page_blocks, int num_pages, int budget, int recent,
                                                                 int first, int longest, int cluster, int room) {
  extern __shared__ uint32_t kept_keys[];
  __shared__ __align__(16) uint32_t hist[3][kDigits], totals[4];
  __shared__ uint32_t scratch[kEvictWarps], chosen[2], warp_counts[2 * kEvictWarps], source[kMoveRows], target[kMoveRows];
  __shared__ uint8_t source_row[kMoveRows];
  ts_pdl_prologue();
  const int rank = blockIdx.x % cluster, head = blockIdx.x / cluster, b = blockIdx.y, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int page_size = page_blocks * KV4_BLOCK;
  const int n = min(context[b], longest);  // (within the block table, and no row that has no place in `order`, whatever the length says)
  if (blockIdx.x == 0 && tid == 0) new_lens[b] = min(n, budget);
  if (n <= budget) return;
  table += (size_t)b * table_stride;
  order += ((size_t)b * nkv + head) * budget;
  auto page_of = [&](int row) { return min(max(table[row / page_size], 0), num_pages - 1); };
  // a row's record among the pool's (its weight then has the place 16 * record + row % 16)
  auto record_of = [&](int row) { return ((uint32_t)page_of(row) * nkv + head) * page_blocks + row % page_size / KV4_BLOCK; };
  auto weight_of = [&](uint32_t record, int row) -> float& { return sums[(size_t)record * KV4_BLOCK + row % KV4_BLOCK]; };

  const int run = ((n + cluster - 1) / cluster + 31) / 32 * 32, row_lo = min(n, rank * run), row_hi = min(n, row_lo + run);
  const bool in_smem = run <= room;
  for (int i = tid; i < 3 * kDigits; i += kEvictThreads) hist[0][i] = 0;
  if (in_smem) {
    constexpr int kAhead = 4;  // loads under way per thread
    for (int i0 = row_lo + tid; i0 < row_hi; i0 += kEvictThreads * kAhead) {
      uint32_t record[kAhead];
      float w[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) record[u] = record_of(min(i0 + u * kEvictThreads, row_hi - 1));
#pragma unroll
      for (int u = 0; u < kAhead; ++u) w[u] = weight_of(record[u], min(i0 + u * kEvictThreads, row_hi - 1));
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i0 + u * kEvictThreads < row_hi) kept_keys[i0 + u * kEvictThreads - row_lo] = order_of(w[u]);
    }
  }
  __syncthreads();
  auto key_of = [&](int i) { return in_smem ? kept_keys[i - row_lo] : order_of(weight_of(record_of(i), i)); };

  uint32_t threshold = 0xffffffffu, ties = 0;  // kept: what is above the threshold, and `ties` of what equals it
  const bool ranked = budget > first + recent;
  if (ranked) {
    uint32_t left = budget - first - recent;  // of the rows [first, n - recent), which are more than that
    threshold = 0;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = max(first, row_lo) + tid; i < min(n - recent, row_hi); i += kEvictThreads) {
        const uint32_t u = key_of(i);
        if (pass == 0 || ((u ^ threshold) >> (shift + bits)) == 0) atomicAdd(&hist[pass][(u >> shift) & ((1u << bits) - 1u)], 1u);
      }
      cluster_meet();
      // the bin in which the count from the top reaches what is left: thread i stands for four bins from 2047 - 4 i down
      constexpr int kBins = kDigits / kEvictThreads;
      static_assert(kBins == 4, "a thread reads its bins at once");
      uint32_t count[kBins] = {0u, 0u, 0u, 0u}, total;
      for (int r = 0; r < cluster; ++r) {
        const uint4 c = peer_words(&hist[pass][kDigits - kBins * (tid + 1)], r);
        count[0] += c.w, count[1] += c.z, count[2] += c.y, count[3] += c.x;
      }
      const uint32_t mine = count[0] + count[1] + count[2] + count[3];
      uint32_t above = block_prefix(mine, scratch, total);
      if (above < left && above + mine >= left) {
#pragma unroll
        for (int j = 0; j < kBins; ++j) {
          if (above < left && above + count[j] >= left) chosen[0] = kDigits - 1 - (tid * kBins + j), chosen[1] = left - above;
          above += count[j];
        }
      }
      __syncthreads();
      threshold |= chosen[0] << shift;
      left = chosen[1];
    }
    ties = left;
  }

  // ---- places: a warp goes over a run of rows, 32 at a time, counting first and then numbering
  auto state_of = [&](int i) -> int {  // 1: kept, 2: of the threshold's own weight
    if (i >= row_hi) return 0;
    if (i < first || i >= n - recent) return 1;
    if (!ranked) return 0;
    const uint32_t u = key_of(i);
    return u > threshold ? 1 : u == threshold ? 2 : 0;
  };
  const int warp_run = (run + kEvictThreads - 1) / kEvictThreads * 32, row0 = row_lo + warp * warp_run, row1 = min(row_hi, row0 + warp_run);
  int sure = 0, equal = 0;
  for (int i = row0; i < row1; i += 32) {
    const int st = state_of(i + lane);
    sure += __popc(__ballot_sync(0xffffffffu, st == 1)), equal += __popc(__ballot_sync(0xffffffffu, st == 2));
  }
  if (lane == 0) warp_counts[warp] = sure, warp_counts[kEvictWarps + warp] = equal;
  __syncthreads();
  if (tid == 0) {
    uint32_t a = 0, e = 0;
    for (int i = 0; i < kEvictWarps; ++i) a += warp_counts[i], e += warp_counts[kEvictWarps + i];
    totals[0] = a, totals[1] = e;
  }
  cluster_meet();
  int sure_before = 0, equal_before = 0;
  for (int r = 0; r < rank; ++r) {
    const uint4 t = peer_words(totals, r);
    sure_before += t.x, equal_before += t.y;
  }
  for (int i = 0; i < warp; ++i) sure_before += warp_counts[i], equal_before += warp_counts[kEvictWarps + i];
  for (int i = row0; i < row1; i += 32) {
    const int row = i + lane, st = state_of(row);
    const uint32_t sures = __ballot_sync(0xffffffffu, st == 1), equals = __ballot_sync(0xffffffffu, st == 2), lower = (1u << lane) - 1u;
    const int e = equal_before + __popc(equals & lower);
    const int place = sure_before + __popc(sures & lower) + min(e, (int)ties);
    if (st == 1 || (st == 2 && e < (int)ties)) __stcg(order + place, row);
    sure_before += __popc(sures), equal_before += __popc(equals);
  }
  cluster_meet();

  // ---- the move: pieces of 16 bytes of codes, pieces of kScale bytes of scales, and the weights
  constexpr int kPieces = D / 16, kCode = kMoveRows * kPieces / kEvictThreads, kScale = D / 16;
  static_assert(kEvictThreads == 2 * kMoveRows, "a thread for the scales of a row's keys, one for its values'");
  const int mine = tid % kMoveRows, half = tid / kMoveRows * (9 * D);
  int coming = rank * kMoveRows + mine < budget ? __ldcg(order + rank * kMoveRows + mine) : 0;  // the source of this thread's place
  for (int base = 0; base < budget; base += kMoveRows * cluster) {
    const int place0 = base + rank * kMoveRows, count = min(max(budget - place0, 0), kMoveRows);
    if (tid < count) {
      source[tid] = record_of(coming), source_row[tid] = coming % KV4_BLOCK;
      target[tid] = record_of(place0 + tid);
    }
    __syncthreads();
    const int next = place0 + kMoveRows * cluster + mine;
    if (next < budget) coming = __ldcg(order + next);
    auto code_at = [&](uint32_t record, int row, int piece) {
      return reinterpret_cast<uint4*>(pool + (size_t)record * (18 * D) + piece / (kPieces / 2) * (9 * D) + row * (D / 2) + piece % (kPieces / 2) * 16);
    };
    auto scale_at = [&](uint32_t record, int row) { return reinterpret_cast<uint32_t*>(pool + (size_t)record * (18 * D) + half + 8 * D + row * kScale); };
    uint4 code[kCode];
    uint32_t scale[kScale / 4];
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < kCode; ++i) {
      const int x = tid + i * kEvictThreads, r = x / kPieces;
      if (r < count) code[i] = *code_at(source[r], source_row[r], x % kPieces);
    }
    if (mine < count) {
#pragma unroll
      for (int i = 0; i < kScale / 4; ++i) scale[i] = scale_at(source[mine], source_row[mine])[i];
      if (half == 0) w = weight_of(source[mine], source_row[mine]);
    }
    cluster_meet();
#pragma unroll
    for (int i = 0; i < kCode; ++i) {
      const int x = tid + i * kEvictThreads, r = x / kPieces;
      if (r < count) *code_at(target[r], (place0 + r) % KV4_BLOCK, x % kPieces) = code[i];
    }
    if (mine < count) {
#pragma unroll
      for (int i = 0; i < kScale / 4; ++i) scale_at(target[mine], (place0 + mine) % KV4_BLOCK)[i] = scale[i];
      if (half == 0) weight_of(target[mine], place0 + mine) = w;
    }
    __syncthreads();
  }
  // (every CTA of the cluster has read all it reads)
  for (int row = budget + rank * kEvictThreads + tid; row < n; row += kEvictThreads * cluster) weight_of(record_of(row), row) = 0.f;
}

template <int D>
int launch_evict(uint8_t* pool, float* sums, const int* table, int table_stride, const int* context, int* new_lens, int* order, int num_seqs, int nkv,
                 int page_blocks, int num_pages, int max_context, int budget, int recent, int first, cudaStream_t stream) {
  static bool set = false;
  if (!set) {
    cudaError_t e = cudaFuncSetAttribute(evict_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeptKeys * 4);
    if (e != cudaSuccess) return (int)e;
    set = true;
  }
  // CTAs per request and head: no more than there are rounds' worth of rows, four where there are few pairs of a request and a head, and eight only
  // where there are very few, for clusters of eight find places late (us with 1 / 2 / 4 / 8: 8 pairs of 40,000 rows 384 / 203 / 79 / 48, 32 of
  // 4,200 51 / 31 / 28 / 44, 64 of 8,190 62 / 46 / 39 / 77, 128 of 8,190 75 / 55 / 41 / 91).
  const long long pairs = (long long)num_seqs * nkv;
  int cluster = 1;
  while (cluster < (pairs <= 16 ? 8 : 4) && cluster * kMoveRows < budget && pairs * cluster < 2 * 148) cluster *= 2;
  const int run = ((max_context + cluster - 1) / cluster + 31) / 32 * 32, room = run < kKeptKeys ? run : kKeptKeys;  // weights in shared memory
  const long long places = (long long)table_stride * page_blocks * KV4_BLOCK;
  const int longest = places < max_context ? (int)places : max_context;
  return ts_launch_cluster(evict_kernel<D>, dim3(nkv * cluster, num_seqs), dim3(kEvictThreads), (size_t)room * 4, stream, cluster, pool, sums, table, table_stride,
                           context, new_lens, order, nkv, page_blocks, num_pages, budget, recent, first, longest, cluster, room);
}

}  // namespace

// Threads per token of the row kernels: with few tokens all groups of a token at once, with many a warp per token.  us a call of 128 / 32 threads, the host's
// part among them, rows of 8 heads of 128: store of 8 tokens 7 / 10, of 1,024 8 / 10, of 4,096 14 / 12; load of 8 6 / 8, of 1,024 8 / 8, of 4,096 14 / 10.
static int threads_per_token(int tokens) { return tokens < 1024 ? 128 : 32; }

// k, v: rows [tokens] of nkv * d entries, `stride` entries apart; slots [tokens], -1: not stored; sums: null or the pool's weights.
// (These entry points take their arguments as one block of memory: a call from Python converts one argument instead of fourteen, which is a
// tenth of what a small call costs the host.)
struct Kv4StoreArgs {
  const void *k, *v;
  long long k_stride, v_stride;
  void* pool;
  float* sums;
  const int* slots;
  void* stream;
  int dtype, tokens, nkv, d, page_blocks, num_pages;
};
TS_EXPORT int ts_kv4_store(const Kv4StoreArgs* args) {
  const auto [k, v, k_stride, v_stride, pool, sums, slots, stream, dtype, tokens, nkv, d, page_blocks, num_pages] = *args;
  if (tokens < 1) return 0;
  const int width = threads_per_token(tokens), log_groups = d == 64 ? 2 : d == 128 ? 3 : 4, num_slots = num_pages * page_blocks * KV4_BLOCK;
  const dim3 grid((unsigned)((tokens + 128 / width - 1) / (128 / width)));
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TS_DTYPE_F32)
    return ts_launch(store_kernel<float>, grid, dim3(128), 0, s, (const float*)k, (const float*)v, k_stride, v_stride, (uint8_t*)pool, sums, slots, tokens,
                     nkv, log_groups, page_blocks, num_slots, width);
  return ts_launch(store_kernel<__nv_bfloat16>, grid, dim3(128), 0, s, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, k_stride, v_stride, (uint8_t*)pool,
                   sums, slots, tokens, nkv, log_groups, page_blocks, num_slots, width);
}

// k, v [rows][nkv][d]; a slot outside the pool gives zeros.
struct Kv4LoadArgs {
  const void* pool;
  const int* slots;
  void *k, *v, *stream;
  int dtype, rows, nkv, d, page_blocks, num_pages;
};
TS_EXPORT int ts_kv4_load(const Kv4LoadArgs* args) {
  const auto [pool, slots, k, v, stream, dtype, rows, nkv, d, page_blocks, num_pages] = *args;
  if (rows < 1) return 0;
  const int width = threads_per_token(rows), log_groups = d == 64 ? 2 : d == 128 ? 3 : 4, num_slots = num_pages * page_blocks * KV4_BLOCK;
  const dim3 grid((unsigned)((rows + 128 / width - 1) / (128 / width)));
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TS_DTYPE_F32)
    return ts_launch(load_kernel<float>, grid, dim3(128), 0, s, (const uint8_t*)pool, slots, (float*)k, (float*)v, rows, nkv, log_groups, page_blocks,
                     num_slots, width);
  return ts_launch(load_kernel<__nv_bfloat16>, grid, dim3(128), 0, s, (const uint8_t*)pool, slots, (__nv_bfloat16*)k, (__nv_bfloat16*)v, rows, nkv,
                   log_groups, page_blocks, num_slots, width);
}

// k, v: [num_seqs * blocks][128][nkv][128] bfloat16, out_table [num_seqs][blocks]; blocks * 128 rows hold the longest request.  out [tokens][nkv * group][128],
// lse and sinks (or null) of as many heads: the attention's, of which the tokens that see nothing are written here.
TS_EXPORT int ts_kv4_expand(const void* pool, const int* table, int table_stride, const int* cu, const int* context, void* k, void* v, int* out_table,
                            int* out_lens, void* out, float* lse, const float* sinks, int num_seqs, int group, int nkv, int page_blocks, int num_pages,
                            int blocks, int window, void* stream) {
  if (num_seqs < 1 || blocks < 1) return 0;
  if (num_seqs > 65535 || nkv > 65535) return TS_ERR_UNSUPPORTED_SIZE;
  return ts_launch(expand_kernel, dim3(blocks * (kExpandPage / kExpandRows), nkv, num_seqs), dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)pool, table,
                   table_stride, cu, context, (uint4*)k, (uint4*)v, out_table, out_lens, (uint4*)out, lse, sinks, group, nkv, page_blocks, num_pages, blocks, window);
}

// order: num_seqs * nkv * budget ints of workspace, none where budget >= max_context; context[b] <= max_context (a longer one counts as that).
struct Kv4EvictArgs {
  void* pool;
  float* sums;
  const int *table, *context;
  int *new_lens, *order;
  void* stream;
  int table_stride, num_seqs, nkv, d, page_blocks, num_pages, max_context, budget, recent, first;
};
TS_EXPORT int ts_kv4_evict(const Kv4EvictArgs* args) {
  const auto [pool, sums, table, context, new_lens, order, stream, table_stride, num_seqs, nkv, d, page_blocks, num_pages, max_context, budget, recent,
              first] = *args;
  if (num_seqs < 1) return 0;
  if (num_seqs > 65535) return TS_ERR_UNSUPPORTED_SIZE;
  if (recent < 0 || first < 0 || budget < 1 || recent + first > budget) return TS_ERR_BAD_ARGUMENT;
  auto launch = d == 64 ? launch_evict<64> : d == 128 ? launch_evict<128> : launch_evict<256>;
  return launch((uint8_t*)pool, sums, table, table_stride, context, new_lens, order, num_seqs, nkv, page_blocks, num_pages, max_context, budget, recent,
                first, (cudaStream_t)stream);
}
