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

// Where the codes and the scales of group `grp` of a row lie.
struct Place {
  size_t codes, scales;
};
__device__ __forceinline__ Place place_of(int slot, int head, int grp, bool values, int nkv, int page_blocks, int d) {
  const int page_size = page_blocks * KV4_BLOCK, page = slot / page_size, row = slot % page_size;
  const size_t rec = (((size_t)page * nkv + head) * page_blocks + row / KV4_BLOCK) * (18 * d) + (values ? 9 * d : 0);
  return {rec + row % KV4_BLOCK * (d / 2) + grp * 8, rec + 8 * d + row % KV4_BLOCK * (d / 16) + grp};
}

// A thread takes the 16 channels of one group: their largest, the scale, the codes, 8 + 1 bytes out.
template <typename T>
__global__ void __launch_bounds__(128) store_kernel(const T* k, const T* v, long long k_stride, long long v_stride, uint8_t* pool, float* sums,
                                                    const int* slots, int tokens, int nkv, int d, int page_blocks, int num_slots) {
  ts_pdl_prologue();
  const int groups = d / 16, per_token = 2 * nkv * groups;
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  const int token = (int)(i / per_token), rest = (int)(i % per_token);
  if (token >= tokens) return;
  const int slot = slots[token];
  if (slot < 0 || slot >= num_slots) return;
  const bool values = rest >= nkv * groups;
  const int unit = rest % (nkv * groups), head = unit / groups, grp = unit % groups;
  float x[16];
  read_group<T>((values ? v + token * v_stride : k + token * k_stride) + unit * 16, x);
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if (x[j] != x[j]) x[j] = 0.f;
    amax = fmaxf(amax, fabsf(x[j]));
  }
  const uint32_t byte = scale_byte(amax);
  const float s = byte ? scale_of(byte) : 1.f;  // (a scale of zero: the whole group rounds to zero)
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int code = byte ? __float2int_rn(fminf(fmaxf(x[j] / s, -7.f), 7.f)) + 8 : 8;
    w[j / 8] |= (uint32_t)code << (4 * (j % 8));
  }
  const Place at = place_of(slot, head, grp, values, nkv, page_blocks, d);
  *reinterpret_cast<uint2*>(pool + at.codes) = make_uint2(w[0], w[1]);
  pool[at.scales] = (uint8_t)byte;
  if (sums != nullptr && !values && grp == 0) {  // a row that comes in has gathered no weight
    const int page_size = page_blocks * KV4_BLOCK;
    sums[((size_t)(slot / page_size) * nkv + head) * page_size + slot % page_size] = 0.f;
  }
}

__device__ __forceinline__ void write_group(float* p, const float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
}
__device__ __forceinline__ void write_group(__nv_bfloat16* p, const float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    __nv_bfloat162 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __floats2bfloat162_rn(x[8 * i + 2 * j], x[8 * i + 2 * j + 1]);
    reinterpret_cast<uint4*>(p)[i] = *reinterpret_cast<const uint4*>(v);
  }
}

template <typename T>
__global__ void __launch_bounds__(128) load_kernel(const uint8_t* pool, const int* slots, T* k, T* v, int rows, int nkv, int d, int page_blocks,
                                                   int num_slots) {
  ts_pdl_prologue();
  const int groups = d / 16, per_row = 2 * nkv * groups;
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  const int row = (int)(i / per_row), rest = (int)(i % per_row);
  if (row >= rows) return;
  const bool values = rest >= nkv * groups;
  const int unit = rest % (nkv * groups);
  const int slot = slots[row];
  float x[16];
  if (slot < 0 || slot >= num_slots) {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = 0.f;
  } else {
    const Place at = place_of(slot, unit / groups, unit % groups, values, nkv, page_blocks, d);
    const uint2 c = *reinterpret_cast<const uint2*>(pool + at.codes);
    const float s = scale_of(pool[at.scales]);
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = (float)((int)(((j < 8 ? c.x : c.y) >> (4 * (j % 8))) & 15u) - 8) * s;
  }
  write_group((values ? v : k) + ((size_t)row * nkv * groups + unit) * 16, x);
}

// The rows that a batch's queries can see, of heads of 128, as bfloat16 pages of 128 rows for the prompt attention, and the block table of those
// pages: request b has the pages [b * blocks, (b + 1) * blocks); out_lens: its rows, as many as have a place.  A CTA unpacks 64 rows of one head.
constexpr int kExpandRows = 64, kExpandPage = 128, kExpandDim = 128;
__global__ void __launch_bounds__(256) expand_kernel(const uint8_t* pool, const int* table, int table_stride, const int* cu, const int* context, uint4* k,
                                                     uint4* v, int* out_table, int* out_lens, int nkv, int page_blocks, int num_pages, int blocks,
                                                     int window) {
  ts_pdl_prologue();
  constexpr int kGroups = kExpandDim / 16, kUnits = kExpandRows * kGroups * 2 / 256;
  const int b = blockIdx.z, head = blockIdx.y, first = blockIdx.x * kExpandRows;
  const int n = min(context[b], min(table_stride * page_blocks * KV4_BLOCK, blocks * kExpandPage));
  if (head == 0 && threadIdx.x == 0) {
    if (first % kExpandPage == 0) out_table[b * blocks + first / kExpandPage] = b * blocks + first / kExpandPage;
    if (first == 0) out_lens[b] = n;
  }
  const int queries = cu[b + 1] - cu[b], oldest = window > 0 ? n - queries - window + 1 : 0;  // the first key that some query sees
  if (first >= n || first + kExpandRows <= oldest || queries <= 0) return;
  uint2 code[kUnits];
  uint32_t scale[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int unit = threadIdx.x + 256 * i, grp = unit % kGroups, values = unit / (kExpandRows * kGroups);
    const int row = min(first + unit / kGroups % kExpandRows, n - 1), blk = row / KV4_BLOCK;
    const int page = min(max(table[(size_t)b * table_stride + blk / page_blocks], 0), num_pages - 1);
    const uint8_t* rec = pool + (((size_t)page * nkv + head) * page_blocks + blk % page_blocks) * (18 * kExpandDim) + values * 9 * kExpandDim;
    code[i] = *reinterpret_cast<const uint2*>(rec + row % KV4_BLOCK * (kExpandDim / 2) + grp * 8);
    scale[i] = rec[8 * kExpandDim + row % KV4_BLOCK * kGroups + grp];
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int unit = threadIdx.x + 256 * i, grp = unit % kGroups, values = unit / (kExpandRows * kGroups);
    const int row = first + unit / kGroups % kExpandRows;
    __nv_bfloat162 f, c;
    kv4_factors(scale[i], scale[i], f, c);
    uint4 out[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t x = j ? code[i].y : code[i].x;
      const uint32_t p0 = kv4_pair(x << 3, f, c), p1 = kv4_pair(x >> 1, f, c), p2 = kv4_pair(x >> 5, f, c), p3 = kv4_pair(x >> 9, f, c);
      out[j] = make_uint4(__byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632), __byte_perm(p2, p3, 0x7632));
    }
    uint4* dst = (values ? v : k) + (((size_t)b * blocks * kExpandPage + row) * nkv + head) * (kExpandDim / 8) + grp * 2;
    if (row < n) dst[0] = out[0], dst[1] = out[1];
  }
}

// ---------------------------------------------------------------------------
// eviction

constexpr int kEvictThreads = 256;

// A weight as an unsigned number of the same order; NaN is the largest, both zeros are one.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sums of both halves of `v` over the threads before this one; `total`: over all of them.
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
  for (int i = 0; i < kEvictThreads / 32; ++i) {
    const uint32_t s = scratch[i];
    if (i < warp) before += s;
    all += s;
  }
  __syncthreads();
  total = all;
  return before + x - v;
}

// One CTA per request and head.  The weights between the first and the recent rows are ranked by a radix select
// (four passes over 8 bits each, from the top); then the rows are gone through in order, 256 at a time, and the kept
// ones move forward.  A row never moves backwards, and what a chunk writes lies before everything that later chunks
// read, so one barrier between a chunk's reads and its writes makes the move safe in place.
__global__ void __launch_bounds__(kEvictThreads) evict_kernel(uint8_t* pool, float* sums, const int* table, int table_stride, const int* context,
                                                              int* new_lens, int nkv, int d, int page_blocks, int num_pages, int budget, int recent,
                                                              int first) {
  __shared__ uint32_t hist[256], scratch[kEvictThreads / 32], chosen[2], list[kEvictThreads];
  ts_pdl_prologue();
  const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int page_size = page_blocks * KV4_BLOCK;
  const int n = min(context[b], table_stride * page_size);
  if (head == 0 && tid == 0) new_lens[b] = min(n, budget);
  if (n <= budget) return;
  table += (size_t)b * table_stride;
  auto page_of = [&](int row) { return min(max(table[row / page_size], 0), num_pages - 1); };
  auto weight_at = [&](int row) -> float& { return sums[((size_t)page_of(row) * nkv + head) * page_size + row % page_size]; };

  uint32_t threshold = 0, ties = 0;
  {
    uint32_t left = budget - first - recent;  // of the rows [first, n - recent), which are more than that
    if (left == 0) {
      threshold = 0xffffffffu;  // nothing passes it, and no tie is taken
    } else {
      for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kEvictThreads) hist[i] = 0;
        __syncthreads();
        for (int i = first + tid; i < n - recent; i += kEvictThreads) {
          const uint32_t u = order_of(weight_at(i));
          if (shift == 24 || (u >> (shift + 8)) == (threshold >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255u], 1u);
        }
        __syncthreads();
        // the bin in which the count from the top reaches what is left: thread i stands for bin 255 - i
        uint32_t total;
        const uint32_t mine = hist[255 - tid];
        const uint32_t above = block_prefix(mine, scratch, total);
        if (above < left && above + mine >= left) chosen[0] = 255 - tid, chosen[1] = left - above;
        __syncthreads();
        threshold |= chosen[0] << shift;
        left = chosen[1];
        __syncthreads();
      }
      ties = left;
    }
  }

  const int row_words = 9 * d / 32;  // of 4 bytes: key codes, key scales, value codes, value scales
  const int code_words = d / 8, scale_words = d / 64;
  auto word_at = [&](int row, int w) {
    uint8_t* rec = pool + (((size_t)page_of(row) * nkv + head) * page_blocks + row % page_size / KV4_BLOCK) * (18 * d);
    const int r = row % KV4_BLOCK, half = code_words + scale_words;
    if (w >= half) w -= half, rec += 9 * d;
    return reinterpret_cast<uint32_t*>(w < code_words ? rec + r * (d / 2) + 4 * w : rec + 8 * d + r * (d / 16) + 4 * (w - code_words));
  };
  int out = 0;
  for (int base = 0; base < n; base += kEvictThreads) {
    const int row = base + tid;
    float w = 0.f;
    uint32_t flag = 0;  // low half: kept for certain, high half: of the threshold's own weight
    if (row < n) {
      w = weight_at(row);
      const uint32_t u = order_of(w);
      if (row < first || row >= n - recent) flag = 1u;
      else if (budget > first + recent) flag = u > threshold ? 1u : u == threshold ? 0x10000u : 0u;
    }
    uint32_t total;
    const uint32_t before = block_prefix(flag, scratch, total);
    const uint32_t ties_before = min(before >> 16, ties);
    const bool keep = (flag & 1u) || (flag && (before >> 16) < ties);
    const int place = (int)((before & 0xffffu) + ties_before);
    const int count = (int)((total & 0xffffu) + min(total >> 16, ties));
    if (keep) {
      list[place] = row;
      weight_at(out + place) = w;
    }
    ties -= min(total >> 16, ties);
    __syncthreads();
    constexpr int kHold = 12;
    for (int at = 0; at < count * row_words; at += kEvictThreads * kHold) {
      uint32_t hold[kHold];
#pragma unroll
      for (int i = 0; i < kHold; ++i) {
        const int x = at + i * kEvictThreads + tid;
        if (x < count * row_words) hold[i] = *word_at(list[x / row_words], x % row_words);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kHold; ++i) {
        const int x = at + i * kEvictThreads + tid;
        if (x < count * row_words) *word_at(out + x / row_words, x % row_words) = hold[i];
      }
    }
    out += count;
    __syncthreads();
  }
  for (int row = out + tid; row < n; row += kEvictThreads) weight_at(row) = 0.f;
}

}  // namespace

// k, v: rows [tokens] of nkv * d entries, `stride` entries apart; slots [tokens], -1: not stored; sums: null or the pool's weights.
TS_EXPORT int ts_kv4_store(const void* k, const void* v, int dtype, long long k_stride, long long v_stride, void* pool, float* sums, const int* slots,
                           int tokens, int nkv, int d, int page_blocks, int num_pages, void* stream) {
  if (tokens < 1) return 0;
  const long long threads = (long long)tokens * 2 * nkv * (d / 16);
  const dim3 grid((unsigned)((threads + 127) / 128));
  const int num_slots = num_pages * page_blocks * KV4_BLOCK;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TS_DTYPE_F32)
    return ts_launch(store_kernel<float>, grid, dim3(128), 0, s, (const float*)k, (const float*)v, k_stride, v_stride, (uint8_t*)pool, sums, slots, tokens,
                     nkv, d, page_blocks, num_slots);
  return ts_launch(store_kernel<__nv_bfloat16>, grid, dim3(128), 0, s, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, k_stride, v_stride, (uint8_t*)pool,
                   sums, slots, tokens, nkv, d, page_blocks, num_slots);
}

// k, v [rows][nkv][d]; a slot outside the pool gives zeros.
TS_EXPORT int ts_kv4_load(const void* pool, const int* slots, void* k, void* v, int dtype, int rows, int nkv, int d, int page_blocks, int num_pages,
                          void* stream) {
  if (rows < 1) return 0;
  const long long threads = (long long)rows * 2 * nkv * (d / 16);
  const dim3 grid((unsigned)((threads + 127) / 128));
  const int num_slots = num_pages * page_blocks * KV4_BLOCK;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TS_DTYPE_F32)
    return ts_launch(load_kernel<float>, grid, dim3(128), 0, s, (const uint8_t*)pool, slots, (float*)k, (float*)v, rows, nkv, d, page_blocks, num_slots);
  return ts_launch(load_kernel<__nv_bfloat16>, grid, dim3(128), 0, s, (const uint8_t*)pool, slots, (__nv_bfloat16*)k, (__nv_bfloat16*)v, rows, nkv, d,
                   page_blocks, num_slots);
}

// k, v: [num_seqs * blocks][128][nkv][128] bfloat16, out_table [num_seqs][blocks]; blocks * 128 rows hold the longest request.
TS_EXPORT int ts_kv4_expand(const void* pool, const int* table, int table_stride, const int* cu, const int* context, void* k, void* v, int* out_table,
                            int* out_lens, int num_seqs, int nkv, int page_blocks, int num_pages, int blocks, int window, void* stream) {
  if (num_seqs < 1 || blocks < 1) return 0;
  if (num_seqs > 65535 || nkv > 65535) return TS_ERR_UNSUPPORTED_SIZE;
  return ts_launch(expand_kernel, dim3(blocks * (kExpandPage / kExpandRows), nkv, num_seqs), dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)pool, table,
                   table_stride, cu, context, (uint4*)k, (uint4*)v, out_table, out_lens, nkv, page_blocks, num_pages, blocks, window);
}

TS_EXPORT int ts_kv4_evict(void* pool, float* sums, const int* table, int table_stride, const int* context, int* new_lens, int num_seqs, int nkv, int d,
                           int page_blocks, int num_pages, int budget, int recent, int first, void* stream) {
  if (num_seqs < 1) return 0;
  if (num_seqs > 65535) return TS_ERR_UNSUPPORTED_SIZE;
  if (recent < 0 || first < 0 || budget < 1 || recent + first > budget) return TS_ERR_BAD_ARGUMENT;
  return ts_launch(evict_kernel, dim3(nkv, num_seqs), dim3(kEvictThreads), 0, (cudaStream_t)stream, (uint8_t*)pool, sums, table, table_stride, context,
                   new_lens, nkv, d, page_blocks, num_pages, budget, recent, first);
}
