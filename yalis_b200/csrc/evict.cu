// Eviction from a paged cache by a running sum per token and KV head.
//
// Of the L tokens of a request, every KV head keeps the last `recent` and, of the others, the keep - recent with the largest sums
// (equal ones: the earlier; NaN counts below everything); they move to the front of the request's pages in their order, sums and
// rows of every pool alike.  Requests of at most `keep` tokens stay as they are.
//
// A block per (request, KV head).  Choice: the sums as ordered 32-bit keys, the border by four histograms of eight bits each, then
// one walk that numbers what stays (a sum over the block per step).  Move: the j-th row that stays lies at or behind place j, so
// in rounds of consecutive rows (all of them read, the block meets, all written) no row is overwritten before it was read.
// Bound by memory: the sums are read six times (L2), a row that moves is read and written once.
#include "common.cuh"

namespace {

constexpr int kThreads = 1024;
constexpr int kPools = 4;
constexpr int kRound = 4;      // units of 16 (or 4, 2) bytes that a thread holds between reading and writing

struct EvictParams {
  unsigned char* pool[kPools];
  int row_bytes[kPools], unit[kPools];     // unit: 16, 4 or 2 bytes a copy
  int n_pools;
  float* sums;                 // [pages, g, page_size]
  const int32_t* lengths;      // [R]
  const int32_t* block_table;  // [R, table_width]
  int table_width, page_size, num_pages, g, keep, recent;
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
  int page_size, g, kvh;
  __device__ __forceinline__ size_t at(int token) const {
    const int index = token / page_size;
    return ((size_t)table_row[index] * g + kvh) * page_size + (token - index * page_size);
  }
};

template <typename U>
__device__ __forceinline__ void move_rows(unsigned char* pool, int row_bytes, const Rows& rows, const int32_t* kept, int first, int keep) {
  const int per_row = row_bytes / (int)sizeof(U), total = (keep - first) * per_row;
  U* base = reinterpret_cast<U*>(pool);
  for (int i0 = 0; i0 < total; i0 += kThreads * kRound) {
    U held[kRound];
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      const int i = i0 + u * kThreads + (int)threadIdx.x;
      if (i < total) {
        const int j = i / per_row;
        held[u] = base[rows.at(kept[first + j]) * per_row + (i - j * per_row)];
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      const int i = i0 + u * kThreads + (int)threadIdx.x;
      if (i < total) {
        const int j = i / per_row;
        base[rows.at(first + j) * per_row + (i - j * per_row)] = held[u];
      }
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads, 1) evict_tokens_kernel(const EvictParams p) {
  __shared__ int histogram[256], warp_above[32], warp_equal[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left, s_bad, s_first;
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.x, req = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int length = p.lengths[req];
  int32_t* kept = p.kept + ((size_t)req * p.g + kvh) * p.keep;
  if (length <= p.keep) {
    for (int j = tid; j < p.keep; j += kThreads) kept[j] = j < length ? j : -1;
    return;
  }
  const Rows rows = {p.block_table + (size_t)req * p.table_width, p.page_size, p.g, kvh};
  if (tid == 0) { s_bad = 0; s_prefix = 0u; s_left = p.keep - p.recent; s_first = p.keep; }
  __syncthreads();
  const int pages = (length - 1) / p.page_size + 1;
  for (int i = tid; i < pages; i += kThreads) {
    const int page = i < p.table_width ? rows.table_row[i] : -1;
    if (page < 0 || page >= p.num_pages) s_bad = 1;
  }
  __syncthreads();
  if (s_bad) {                                   // a token without a page: this request stays as it is
    if (tid == 0 && p.error) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);
    for (int j = tid; j < p.keep; j += kThreads) kept[j] = -1;
    return;
  }
  const int others = length - p.recent;          // tokens that are chosen by their sums
  // The border: the s_left-th largest key, eight bits at a time from the top.
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) histogram[i] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
    for (int t = tid; t < others; t += kThreads) {
      const uint32_t key = key_of(p.sums[rows.at(t)]);
      if ((key & mask) == prefix) atomicAdd(&histogram[(key >> shift) & 255u], 1);
    }
    __syncthreads();
    if (warp == 0) {                             // lane 0 holds the largest bins
      int bins[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += bins[i] = histogram[255 - lane * 8 - i];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int below = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += below;
      }
      int above = upto - sum;
      const int left = s_left;
      __syncwarp();
      if (above < left && left <= upto) {        // (one lane; none where nothing is left to choose)
        int i = 0;
        while (above + bins[i] < left) above += bins[i++];
        s_prefix = prefix | (uint32_t)(255 - lane * 8 - i) << shift;
        s_left = left - above;
      }
    }
    __syncthreads();
  }
  const uint32_t border = s_prefix;
  const int take_equal = p.keep == p.recent ? 0 : s_left;      // of the tokens on the border, the earliest
  const bool choose = p.keep > p.recent;
  // What stays, in order.
  int n_kept = 0, n_equal = 0;
  for (int t0 = 0; t0 < length; t0 += kThreads) {
    const int t = t0 + tid;
    bool above = t < length && t >= others, equal = false;
    if (t < others && choose) {
      const uint32_t key = key_of(p.sums[rows.at(t)]);
      above = key > border;
      equal = key == border;
    }
    const unsigned equals = __ballot_sync(0xffffffffu, equal);
    if (lane == 0) warp_equal[warp] = __popc(equals);
    __syncthreads();
    int before = n_equal, all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += warp_equal[w];
      all += warp_equal[w];
    }
    n_equal += all;
    const bool stays = above || (equal && before + __popc(equals & ((1u << lane) - 1u)) < take_equal);
    const unsigned staying = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) warp_above[warp] = __popc(staying);
    __syncthreads();
    int place = n_kept + __popc(staying & ((1u << lane) - 1u));
    all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) place += warp_above[w];
      all += warp_above[w];
    }
    n_kept += all;
    if (stays) {
      kept[place] = t;
      if (place != t) atomicMin(&s_first, place);               // rows before this one are where they belong
    }
    __syncthreads();
  }
  const int first = s_first;
  move_rows<uint32_t>(reinterpret_cast<unsigned char*>(p.sums), 4, rows, kept, first, p.keep);
  for (int i = 0; i < p.n_pools; ++i) {
    if (p.unit[i] == 16) move_rows<uint4>(p.pool[i], p.row_bytes[i], rows, kept, first, p.keep);
    else if (p.unit[i] == 4) move_rows<uint32_t>(p.pool[i], p.row_bytes[i], rows, kept, first, p.keep);
    else move_rows<uint16_t>(p.pool[i], p.row_bytes[i], rows, kept, first, p.keep);
  }
}

}  // namespace

YALIS_API int yalis_evict_tokens(void* const* pools, const int* row_bytes, int n_pools, float* sums, const int32_t* lengths,
                                 const int32_t* block_table, int table_width, int page_size, int num_pages, int g, int n_requests,
                                 int keep, int recent, int32_t* kept, int32_t* error, cudaStream_t stream) {
  if (n_pools < 0 || n_pools > kPools || keep < 1 || recent < 0 || recent > keep || page_size < 1 || g < 1 || n_requests > 65535)
    return YALIS_ERR_SHAPE;
  if (n_requests <= 0) return YALIS_OK;
  EvictParams p = {};
  for (int i = 0; i < n_pools; ++i) {
    p.pool[i] = static_cast<unsigned char*>(pools[i]);
    p.row_bytes[i] = row_bytes[i];
    const uintptr_t both = reinterpret_cast<uintptr_t>(pools[i]) | (uintptr_t)row_bytes[i];
    p.unit[i] = both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : 2;
    if (both % 2) return YALIS_ERR_ALIGN;
  }
  p.n_pools = n_pools; p.sums = sums; p.lengths = lengths; p.block_table = block_table; p.table_width = table_width;
  p.page_size = page_size; p.num_pages = num_pages; p.g = g; p.keep = keep; p.recent = recent; p.kept = kept; p.error = error;
  return yalis_launch(evict_tokens_kernel, dim3(g, n_requests), dim3(kThreads), 0, stream, p);
}
