// Eviction from a paged cache by a running sum per token and KV head.
//
// Of the L tokens of a request, every KV head keeps the last `recent` and, of the others, the keep - recent with the largest sums
// (equal ones: the earlier; NaN counts below everything); they move to the front of the request's pages in their order, sums and
// rows of every pool alike.  Requests of at most `keep` tokens stay as they are.
//
// A block per (request, KV head).  Choice: the sums as ordered 32-bit keys (in shared memory where they fit), the border by three
// histograms of eleven bits and ten, then one walk that numbers what stays, four tokens a thread.  Move: the j-th row that stays lies
// at or behind place j, so in rounds of consecutive rows (all of them read, the block meets, all written) no row is overwritten before
// it was read; a group of lanes takes a row of all pools at once, several rows under way.
// Bound by memory: the sums are read once, a row that moves is read and written once (32 requests of 2,176 to 4,160 tokens to 2,048, 8 KV
// heads of 128 in bfloat16: 101 us, 495 MB at 4.9 TB/s; with nothing to move 27; one request of 700 tokens: 12 us).  A request alone has a
// block for each of its KV heads and nothing for the other SMs: 32,000 tokens to 16,000, 8 KV heads of 128: 710 us in bfloat16 and 308
// in 4 bits, for 20 and 5.5 at the copy's rate; 128,000 to 64,000: 2,850 and 1,240.
#include "common.cuh"
#include "slots.cuh"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kPools = 4;
constexpr int kBins = 2048;
constexpr int kEach = 4;       // neighbouring tokens of a thread in the last walk

struct EvictParams {
  unsigned char* pool[kPools];
  int row_bytes[kPools], unit[kPools];     // unit: 16, 4 or 2 bytes a copy
  int n_pools, lanes;          // lanes: of a group that moves a row (a power of two up to 32)
  float* sums;                 // [pages, g, page_size]
  const int32_t* lengths;      // [R]
  const int32_t* block_table;  // [R, table_width]
  int table_width, page_size, shift, num_pages, g, keep, recent;
  int room;                    // keys that shared memory holds
  int32_t* kept;               // [R, g, keep]
  int32_t* error;
};

// Larger sums have larger keys; NaN has the least.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0u;
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);       // (-0 and 0 are equal)
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

struct Rows {
  const int32_t* table_row;
  int page_size, shift, g, kvh;
  __device__ __forceinline__ size_t at(int token) const {
    const int index = shift >= 0 ? token >> shift : token / page_size;
    return ((size_t)table_row[index] * g + kvh) * page_size + (token - index * page_size);
  }
};

// The sum over the block's threads before this one, and of all of them; `scratch` [kWarps] may be used again after two meetings.
__device__ __forceinline__ int before_in_block(int v, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int below = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += below;
  }
  if (lane == 31) scratch[warp] = upto;
  __syncthreads();
  int mine = lane < kWarps ? scratch[lane] : 0, sums = mine;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const int below = __shfl_up_sync(0xffffffffu, sums, o);
    if (lane >= o) sums += below;
  }
  total = __shfl_sync(0xffffffffu, sums, kWarps - 1);
  return __shfl_sync(0xffffffffu, sums - mine, warp) + upto - v;
}

__device__ __forceinline__ uint4 load_unit(const unsigned char* at, int unit) {
  if (unit == 16) return *reinterpret_cast<const uint4*>(at);
  return make_uint4(unit == 4 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at), 0u, 0u, 0u);
}
__device__ __forceinline__ void store_unit(unsigned char* at, int unit, uint4 v) {
  if (unit == 16) *reinterpret_cast<uint4*>(at) = v;
  else if (unit == 4) *reinterpret_cast<uint32_t*>(at) = v.x;
  else *reinterpret_cast<uint16_t*>(at) = (uint16_t)v.x;
}

// Moves rows kept[first ... keep - 1] to places first ... in pools [P0, P0 + NP), U rows of a group of lanes at a time.
template <int NP, int U, typename Kept>
__device__ __forceinline__ void move_rows(const EvictParams& p, int p0, const Rows& rows, const Kept& kept, int first) {
  const int lane = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes, groups = kThreads / p.lanes;
  int widest = p0 == 0;                                       // pieces of a row that its lanes take in turn (the sums move with the first)
#pragma unroll
  for (int i = 0; i < NP; ++i) widest = max(widest, (p.row_bytes[p0 + i] + p.unit[p0 + i] * p.lanes - 1) / (p.unit[p0 + i] * p.lanes));
  for (int j0 = first; j0 < p.keep; j0 += groups * U) {
    for (int piece = 0; piece < widest; ++piece) {
      uint4 held[U][NP];
      float sum[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * groups + group;
        if (j >= p.keep) break;
        const size_t from = rows.at(kept(j));
        if (p0 == 0 && piece == 0 && lane == 0) sum[u] = p.sums[from];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int byte = (piece * p.lanes + lane) * p.unit[p0 + i];
          if (byte < p.row_bytes[p0 + i]) held[u][i] = load_unit(p.pool[p0 + i] + from * p.row_bytes[p0 + i] + byte, p.unit[p0 + i]);
        }
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * groups + group;
        if (j >= p.keep) break;
        const size_t to = rows.at(j);
        if (p0 == 0 && piece == 0 && lane == 0) p.sums[to] = sum[u];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int byte = (piece * p.lanes + lane) * p.unit[p0 + i];
          if (byte < p.row_bytes[p0 + i]) store_unit(p.pool[p0 + i] + to * p.row_bytes[p0 + i] + byte, p.unit[p0 + i], held[u][i]);
        }
      }
      // (the next round reads rows behind those written here: it need not wait)
    }
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kThreads, 2) evict_tokens_kernel(const EvictParams p) {
  extern __shared__ uint32_t keys[];                          // [room] keys, later the places of what stays
  __shared__ int histogram[kBins], scan[2][kWarps];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left, s_bad, s_first;
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.x, req = blockIdx.y, tid = threadIdx.x;
  const int length = p.lengths[req];
  int32_t* kept = p.kept + ((size_t)req * p.g + kvh) * p.keep;
  if (length <= p.keep) {
    for (int j = tid; j < p.keep; j += kThreads) kept[j] = j < length ? j : -1;
    return;
  }
  const Rows rows = {p.block_table + (size_t)req * p.table_width, p.page_size, p.shift, p.g, kvh};
  if (tid == 0) { s_bad = 0; s_prefix = 0u; s_left = p.keep - p.recent; s_first = p.keep; }
  __syncthreads();
  const int pages = (length - 1) / p.page_size + 1;
  for (int i = tid; i < pages; i += kThreads) {
    const int page = i < p.table_width ? rows.table_row[i] : -1;
    if (page < 0 || page >= p.num_pages) s_bad = 1;
  }
  for (int i = tid; i < kBins; i += kThreads) histogram[i] = 0;
  __syncthreads();
  if (s_bad) {                                   // a token without a page: this request stays as it is
    if (tid == 0 && p.error) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);
    for (int j = tid; j < p.keep; j += kThreads) kept[j] = -1;
    return;
  }
  const int others = length - p.recent;          // tokens that are chosen by their sums
  const bool choose = p.keep > p.recent, here = length <= p.room;
  auto key_at = [&](int t) { return here ? keys[t] : key_of(p.sums[rows.at(t)]); };
  // The border: the s_left-th largest key, eleven bits at a time from the top (the last time ten).
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass < 2 ? 2048 : 1024;
    const uint32_t prefix = s_prefix, mask = pass == 0 ? 0u : 0xFFFFFFFFu << (pass == 1 ? 21 : 10);
    for (int t = tid; t < others; t += kThreads) {
      uint32_t key;
      if (pass == 0 && here) keys[t] = key = key_of(p.sums[rows.at(t)]);
      else key = key_at(t);
      if (choose && (key & mask) == prefix) atomicAdd(&histogram[(key >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    if (!choose) break;
    // Thread i holds the bins from the top down, bins / kThreads of them.
    const int each = bins / kThreads;
    int held[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      held[i] = i < each ? histogram[bins - 1 - tid * each - i] : 0;
      sum += held[i];
    }
    int total, above = before_in_block(sum, scan[pass & 1], total);
    const int left = s_left;
    __syncthreads();                             // (everyone has the bins and what was left)
    for (int i = tid; i < kBins; i += kThreads) histogram[i] = 0;
    if (above < left && left <= above + sum) {   // one thread
      int i = 0;
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (i == k && above + held[k] < left) above += held[k], ++i;
      s_prefix = prefix | (uint32_t)(bins - 1 - tid * each - i) << shift;
      s_left = left - above;
    }
    __syncthreads();
  }
  const uint32_t border = s_prefix;
  const int take_equal = s_left;                 // of the tokens on the border, the earliest
  // What stays, in order.
  int n_kept = 0, n_equal = 0;
  for (int t0 = 0; t0 < length; t0 += kThreads * kEach) {
    const int t = t0 + tid * kEach;
    unsigned above = 0, equal = 0;               // a bit a token
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (t + i >= length) break;
      if (t + i >= others) {
        above |= 1u << i;
      } else if (choose) {
        const uint32_t key = key_at(t + i);
        above |= (unsigned)(key > border) << i;
        equal |= (unsigned)(key == border) << i;
      }
    }
    int all;
    int before = n_equal + before_in_block(__popc(equal), scan[0], all);
    n_equal += all;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (equal >> i & 1u) above |= (unsigned)(before++ < take_equal) << i;
    int place = n_kept + before_in_block(__popc(above), scan[1], all);
    n_kept += all;
    // (every key of this stretch is in a register by now, and places are no further on than tokens: they may take the keys' room)
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (above >> i & 1u) {
        kept[place] = t + i;
        if (here) keys[place] = (uint32_t)(t + i);
        if (place != t + i) atomicMin(&s_first, place);       // rows before this one are where they belong
        ++place;
      }
    __syncthreads();
  }
  const int first = s_first;
  auto source = [&](int j) { return here ? (int)keys[j] : kept[j]; };
  // More rows under way where fewer pools share the registers.
  if (p.n_pools <= 2) move_rows<2, 4>(p, 0, rows, source, first);
  else move_rows<4, 2>(p, 0, rows, source, first);
}

}  // namespace

YALIS_API int yalis_evict_tokens(void* const* pools, const int* row_bytes, int n_pools, float* sums, const int32_t* lengths,
                                 const int32_t* block_table, int table_width, int page_size, int num_pages, int g, int n_requests,
                                 int keep, int recent, int32_t* kept, int32_t* error, cudaStream_t stream) {
  if (n_pools < 0 || n_pools > kPools || keep < 1 || recent < 0 || recent > keep || page_size < 1 || g < 1 || n_requests > 65535)
    return YALIS_ERR_SHAPE;
  if (n_requests <= 0) return YALIS_OK;
  EvictParams p = {};
  int units = 1;
  for (int i = 0; i < kPools; ++i) {
    p.unit[i] = 16;                              // (a pool that is not there has rows of no bytes)
    if (i >= n_pools) continue;
    p.pool[i] = static_cast<unsigned char*>(pools[i]);
    p.row_bytes[i] = row_bytes[i];
    const uintptr_t both = reinterpret_cast<uintptr_t>(pools[i]) | (uintptr_t)row_bytes[i];
    p.unit[i] = both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : 2;
    if (both % 2) return YALIS_ERR_ALIGN;
    if (row_bytes[i] / p.unit[i] > units) units = row_bytes[i] / p.unit[i];
  }
  for (p.lanes = 1; p.lanes < 32 && p.lanes < units;) p.lanes *= 2;
  p.n_pools = n_pools; p.sums = sums; p.lengths = lengths; p.block_table = block_table; p.table_width = table_width;
  p.page_size = page_size; p.num_pages = num_pages; p.g = g; p.keep = keep; p.recent = recent; p.kept = kept; p.error = error;
  while (1 << p.shift < page_size) ++p.shift;
  if (1 << p.shift != page_size) p.shift = -1;
  // Keys of as many tokens as two blocks an SM have room for.
  const long long most = (long long)table_width * page_size;
  p.room = (int)(most < 24 * 1024 ? most : 24 * 1024);
  const int smem = p.room * 4;
  static int configured[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return YALIS_ERR_LAUNCH;
  if (smem > 32 * 1024 && (dev < 0 || dev >= 64 || !configured[dev])) {
    if (cudaFuncSetAttribute(evict_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 24 * 1024 * 4) != cudaSuccess) return YALIS_ERR_LAUNCH;
    if (dev >= 0 && dev < 64) configured[dev] = 1;
  }
  return yalis_launch(evict_tokens_kernel, dim3(g, n_requests), dim3(kThreads), smem, stream, p);
}

YALIS_SLOTS(yalis_evict_tokens)
