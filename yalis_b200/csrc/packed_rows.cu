// Rows of keys and values into pages held in 4 bits, and back.
//
// A row of one token and KV head is taken by dim / 8 neighbouring lanes (a group of 4, 8, 16 or 32), eight values a lane: the
// row's extremes by shuffles, then every lane its word of eight codes.  A block takes rows of one token (keys and values are rows
// of one list), so that the token's place is looked up without a division a thread; of many tokens it takes TOKENS side by side, whose
// look-ups (token, page, row: three trips to memory one after the other) overlap.
// 2 dim values read and dim + 4 bytes written a token and KV head (bfloat16: 512 -> 132 B at 128).  Bound by instructions: 10,002 tokens,
// 8 KV heads of 128 (51.5 MB): 25 us to write (2.1 TB/s, issue slots busy 0.78), 14 to read back (3.7 TB/s, 0.70).
#include "packed.cuh"
#include "slots.cuh"

namespace {

template <typename T>
struct RowParams {
  const T* k;                  // [N, k_stride]
  const T* v;
  long long k_stride, v_stride;
  T* k_out;                    // read: contiguous [N, g * dim]
  T* v_out;
  const int32_t* positions;    // [N] place of the token in its request's cache
  const int32_t* req_of_token; // [N] row of the block table, -1: not a token
  const int32_t* block_table;
  int table_width, n_tokens;
  int vector;                  // 1: rows start on boundaries of 16 bytes
  int32_t* error;
  PackedPages pages;
};

// Eight values of a row as they lie in memory: bfloat16 in pairs, or float32.
struct Pairs { uint32_t w[4]; };
struct Singles { float v[8]; };
template <typename T> struct Held;
template <> struct Held<__nv_bfloat16> { using type = Pairs; };
template <> struct Held<float> { using type = Singles; };

__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool vector, Pairs& x) {
  if (vector) {
    *reinterpret_cast<uint4*>(x.w) = *reinterpret_cast<const uint4*>(p);
  } else {
    const uint16_t* at = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x.w[i] = at[2 * i] | (uint32_t)at[2 * i + 1] << 16;
  }
}
__device__ __forceinline__ void load8(const float* p, bool vector, Singles& x) {
  if (vector) {
    *reinterpret_cast<float4*>(x.v) = load4_f32(p);
    *reinterpret_cast<float4*>(x.v + 4) = load4_f32(p + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = p[i];
  }
}
__device__ __forceinline__ void zero8(Pairs& x) { x.w[0] = x.w[1] = x.w[2] = x.w[3] = 0u; }
__device__ __forceinline__ void zero8(Singles& x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x.v[i] = 0.f;
}
__device__ __forceinline__ void values8(const Pairs& x, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(x.w[i] << 16);
    v[2 * i + 1] = __uint_as_float(x.w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void values8(const Singles& x, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = x.v[i];
}

// The largest of the row's values and 0, and minus the least of them and 0, over LANES neighbouring lanes.
__device__ __forceinline__ uint32_t most2(uint32_t a, uint32_t b) {           // of each half; not a number if one is none
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <int LANES>
__device__ __forceinline__ void extremes(const Pairs& x, float& above, float& below) {
  // both extremes as one pair: the values' largest beside the largest of the values with their signs turned
  const uint32_t sign = 0x80008000u;
  const uint32_t up = most2(most2(x.w[0], x.w[1]), most2(x.w[2], x.w[3]));
  const uint32_t down = most2(most2(x.w[0] ^ sign, x.w[1] ^ sign), most2(x.w[2] ^ sign, x.w[3] ^ sign));
  uint32_t both = most2(most2(__byte_perm(up, down, 0x5410), __byte_perm(up, down, 0x7632)), 0u);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) both = most2(both, __shfl_xor_sync(0xffffffffu, both, o));
  above = __uint_as_float(both << 16);
  below = __uint_as_float(both & 0xFFFF0000u);
}
template <int LANES>
__device__ __forceinline__ void extremes(const Singles& x, float& above, float& below) {
  float odd = 0.f;
  above = below = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    above = fmaxf(above, x.v[i]);
    below = fmaxf(below, -x.v[i]);
    odd = fmaf(x.v[i], 0.f, odd);                             // not a number where a value is none, or infinite
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    above = fmaxf(above, __shfl_xor_sync(0xffffffffu, above, o));
    below = fmaxf(below, __shfl_xor_sync(0xffffffffu, below, o));
    odd += __shfl_xor_sync(0xffffffffu, odd, o);
  }
  above += odd;
}

// The pool's row of a KV head of a token, -1 where the token is none or has no page.
template <typename T>
__device__ __forceinline__ long long place_of(const RowParams<T>& p, int token, int kvh, bool tells) {
  const int req = p.req_of_token[token], at = p.positions[token];
  if (req < 0 || at < 0) return -1;
  int row;
  const int page = page_of(p.pages, p.block_table + (size_t)req * p.table_width, p.table_width, at, row);
  if (page >= 0) return (long long)row_index(p.pages, page, kvh, row);
  if (tells && p.error) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);
  return -1;
}

template <typename T, int LANES, int TOKENS>
__global__ void packed_rows_write_kernel(const RowParams<T> p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & (LANES - 1), group = (blockIdx.y * blockDim.x + threadIdx.x) / LANES, is_v = group & 1, kvh = group >> 1;
  const bool listed = kvh < p.pages.g && lane * 8 < p.pages.dim;
  typename Held<T>::type x[TOKENS];
  long long row[TOKENS];
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    const int token = blockIdx.x * TOKENS + i;
    row[i] = -1;
    zero8(x[i]);
    if (listed && token < p.n_tokens) {
      const T* src = is_v ? p.v + (long long)token * p.v_stride : p.k + (long long)token * p.k_stride;
      load8(src + (size_t)kvh * p.pages.dim + lane * 8, p.vector, x[i]);
      row[i] = place_of(p, token, kvh, group == 0 && lane == 0);
    }
  }
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    float above, below;                                       // the row's extremes, not numbers where it holds one that is none
    extremes<LANES>(x[i], above, below);
    if (row[i] < 0) continue;
    uint32_t codes = 0, word = 0x7FC0u;                       // not a number: all codes 0
    if (above <= kPackedLargest && below <= kPackedLargest) {
      const float step = step_for(below, above);
      float inverse;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(step));
      const float first = multiple_of<sizeof(T) == 4>(-below, step, inverse);
      float v[8];
      values8(x[i], v);
#pragma unroll
      for (int j = 7; j >= 0; --j) {                          // (no value lies below the row's least)
        const int c = __float_as_int(multiple_of<sizeof(T) == 4>(v[j], step, inverse)) - __float_as_int(first);
        codes = codes << 4 | (uint32_t)min(c, 15);
      }
      word = (__float_as_uint(step) >> 16) | (uint32_t)(__float_as_int(12582912.f) - __float_as_int(first));
    }
    (is_v ? p.pages.v : p.pages.k)[row[i] * (p.pages.dim / 8) + lane] = codes;
    if (lane == 0) reinterpret_cast<uint16_t*>(p.pages.words + row[i])[is_v] = (uint16_t)word;
  }
}

template <typename T, int LANES, int TOKENS>
__global__ void packed_rows_read_kernel(const RowParams<T> p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & (LANES - 1), group = (blockIdx.y * blockDim.x + threadIdx.x) / LANES, is_v = group & 1, kvh = group >> 1;
  if (kvh >= p.pages.g || lane * 8 >= p.pages.dim) return;
  long long row[TOKENS];
  uint32_t codes[TOKENS], word[TOKENS];
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    const int token = blockIdx.x * TOKENS + i;
    row[i] = token < p.n_tokens ? place_of(p, token, kvh, group == 0 && lane == 0) : -1;
  }
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    codes[i] = word[i] = 0u;                                  // a token without a page reads as zeros
    if (row[i] >= 0) {
      codes[i] = (is_v ? p.pages.v : p.pages.k)[row[i] * (p.pages.dim / 8) + lane];
      word[i] = reinterpret_cast<const uint16_t*>(p.pages.words + row[i])[is_v];
    }
  }
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    const int token = blockIdx.x * TOKENS + i;
    if (token >= p.n_tokens) return;
    T* dst = (is_v ? p.v_out : p.k_out) + ((size_t)token * p.pages.g + kvh) * p.pages.dim + lane * 8;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(dst) = unpack_bf16(codes[i], word[i]);
    } else {
      const float step = step_of(word[i]), zero = zero_of(word[i]);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = ((float)((codes[i] >> (4 * j)) & 15u) - zero) * step;
      store4(dst, make_float4(x[0], x[1], x[2], x[3]));
      store4(dst + 4, make_float4(x[4], x[5], x[6], x[7]));
    }
  }
}

template <typename T, bool WRITE>
int launch_rows(const RowParams<T>& p, int n_tokens, cudaStream_t stream) {
  const int lanes = p.pages.dim <= 32 ? 4 : p.pages.dim <= 64 ? 8 : p.pages.dim <= 128 ? 16 : 32;
  const long long threads = 2LL * p.pages.g * lanes;          // of a token
  const int block = (int)(threads >= 256 ? 256 : (threads + 31) / 32 * 32);
  const long long per_token = (threads + block - 1) / block;
  if (per_token > 65535) return YALIS_ERR_SHAPE;
  // One token a block while its blocks fit the GPU at once about twice over, else four.
  const bool many = (long long)n_tokens * per_token * block > 4096LL * yalis_sm_count();
  const dim3 grid((unsigned)(many ? (n_tokens + 3) / 4 : n_tokens), (unsigned)per_token);
#define YALIS_ROWS(L)                                                                                                              \
  (many ? yalis_launch(WRITE ? packed_rows_write_kernel<T, L, 4> : packed_rows_read_kernel<T, L, 4>, grid, dim3(block), 0, stream, p) \
        : yalis_launch(WRITE ? packed_rows_write_kernel<T, L, 1> : packed_rows_read_kernel<T, L, 1>, grid, dim3(block), 0, stream, p))
  switch (lanes) {
    case 4: return YALIS_ROWS(4);
    case 8: return YALIS_ROWS(8);
    case 16: return YALIS_ROWS(16);
    default: return YALIS_ROWS(32);
  }
#undef YALIS_ROWS
}

// The visible rows of requests' caches into bfloat16 pools of one call, for kernels that read such pools: pages of kUnpackPage
// keys, request after request (page r * width + i holds keys i * kUnpackPage ... of request r), with the block table that says so
// and the counters of the kernels behind it at zero.  Exact: every value is a bfloat16 number.  A value row without numbers goes in
// as zeros and is marked instead: rows that do not see it give it the weight 0, and 0 times what is no number is none either.  A key
// without a page is zeros and marked too (it would count as a score of 0).
// An item is a page of one KV head; a resident grid walks the items that some request needs, which every block counts for itself
// from the step's lengths (a block for every page that a request could have took 75 us of 64 requests, one of them a portion of
// 4,033 tokens behind 3,967 and the others single tokens behind 8,000 that need none; now 12).  A thread takes eight codes of a row at
// a time.  Bound by the writes (512 B a token and KV head at 128), most of which the reader finds in the L2: 16,384 tokens, 8 KV heads
// of 128, 85 MB: 19 us; of 64: 15 us; 2,048 tokens of 64: 5.6 us (six or eight blocks an SM in place of four: 3 to 14 % slower).
constexpr int kUnpackPage = 64, kUnpackThreads = 256;

struct UnpackParams {
  __nv_bfloat16* k_out;        // [R * width, g, kUnpackPage, dim]
  __nv_bfloat16* v_out;
  uint32_t* marks;             // [R * width, g, 2048 / dim]: of key i + (2048 / dim) j of a page in byte j of word i; of keys that some
                               // row sees, bit 0 where the value holds no numbers, bit 1 where there is no page
  int32_t* some_marked;        // becomes `marked_by`, a number of this launch's own, if any key is marked
  int marked_by;
  int32_t* table_out;          // [R, width]
  int32_t* zeroed;             // [n_zeroed] counters
  int n_zeroed;
  const int32_t* positions;
  const int32_t* q_start;      // [R + 1]
  const int32_t* block_table;
  int table_width, n_requests, width, window, skip_single;
  int32_t* error;
  PackedPages pages;
};

__global__ void __launch_bounds__(kUnpackThreads, 4) packed_unpack_kernel(const UnpackParams p) {
  __shared__ int start[kUnpackThreads + 1], first_key[kUnpackThreads], last_key[kUnpackThreads], warp_sum[kUnpackThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, words = p.pages.dim / 8;
  const long long thread = (long long)blockIdx.x * kUnpackThreads + tid, threads = (long long)gridDim.x * kUnpackThreads;
  for (long long i = thread; i < p.n_zeroed; i += threads) p.zeroed[i] = 0;
  for (long long i = thread; i < (long long)p.n_requests * p.width; i += threads) p.table_out[i] = (int32_t)i;
  // A thread has the same word of codes of every per_round-th row: four rows' look-ups and loads are under way at a time.
  const int w = tid % words, own = tid / words, per_round = kUnpackThreads / words;
  int item = blockIdx.x;                                      // counted from the first item of these requests
  for (int r0 = 0; r0 < p.n_requests; r0 += kUnpackThreads) {
    int pages = 0;
    if (r0 + tid < p.n_requests) {
      const int t0 = p.q_start[r0 + tid], n = p.q_start[r0 + tid + 1] - t0;
      if (n > 1 || (n == 1 && !p.skip_single)) {
        const int place = p.positions[t0 + n - 1], last = min(place, p.width * kUnpackPage - 1);
        if (place > last && blockIdx.x == 0 && p.error) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);       // (it sees places that no pool has)
        const int first = p.window > 0 ? max(0, p.positions[t0] - p.window + 1) : 0;
        first_key[tid] = first;
        last_key[tid] = last;
        if (last >= first) pages = last / kUnpackPage - first / kUnpackPage + 1;
      }
    }
    int sum = pages * p.pages.g;                              // a running sum over the requests
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int before = __shfl_up_sync(0xFFFFFFFFu, sum, d);
      if (lane >= d) sum += before;
    }
    if (lane == 31) warp_sum[tid >> 5] = sum;
    __syncthreads();
    for (int i = 0; i < tid >> 5; ++i) sum += warp_sum[i];
    start[tid + 1] = sum;
    if (tid == 0) start[0] = 0;
    __syncthreads();
    const int total = start[kUnpackThreads];
    for (; item < total; item += gridDim.x) {
      int i = 0;                                              // the request: the last that starts at or before the item
#pragma unroll
      for (int d = kUnpackThreads / 2; d > 0; d >>= 1)
        if (start[i + d] <= item) i += d;
      const int req = r0 + i, local = item - start[i], first = first_key[i], last = last_key[i];
      const int index = first / kUnpackPage + local / p.pages.g, kvh = local % p.pages.g, key0 = index * kUnpackPage;
      const size_t to = (((size_t)req * p.width + index) * p.pages.g + kvh) * kUnpackPage;
      const int32_t* table_row = p.block_table + (size_t)req * p.table_width;
      const int rows = min(kUnpackPage, last - key0 + 1), q = own;        // (four rounds are a page, or two)
      if (q < rows) {
        long long at[4];
        uint32_t word[4], kc[4], vc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = q + j * per_round, key = key0 + r;
          at[j] = -1;
          if (r >= rows) continue;
          int row;
          const int page = page_of(p.pages, table_row, p.table_width, key, row);
          if (page >= 0) at[j] = (long long)row_index(p.pages, page, kvh, row);
          else if (key >= first && w == 0 && p.error) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          word[j] = kc[j] = vc[j] = 0u;
          if (at[j] < 0) continue;
          word[j] = p.pages.words[at[j]];
          kc[j] = p.pages.k[at[j] * words + w];
          vc[j] = p.pages.v[at[j] * words + w];
        }
        uint32_t marked = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = q + j * per_round;
          if (r >= rows) break;
          const bool none = (word[j] >> 16 & 0x7F80u) == 0x7F80u;
          reinterpret_cast<uint4*>(p.k_out)[(to + r) * words + w] = unpack_bf16(kc[j], word[j] & 0xFFFFu);
          reinterpret_cast<uint4*>(p.v_out)[(to + r) * words + w] = unpack_bf16(vc[j], none ? 0u : word[j] >> 16);
          if (key0 + r >= first) marked |= ((none ? 1u : 0u) | (at[j] < 0 ? 2u : 0u)) << (8 * j);       // (pages behind a window may be gone)
        }
        if (w == 0) {
          p.marks[to / kUnpackPage * per_round + q] = marked;
          if (marked) *p.some_marked = p.marked_by;
        }
      }
    }
    item -= total;
    __syncthreads();                                          // (the requests' arrays are written again)
  }
}

}  // namespace

// Writes the rows of n_tokens tokens (write 1), or reads them back into contiguous [N, g * dim] (write 0).
YALIS_API int yalis_packed_rows(int write, void* k, void* v, long long k_stride, long long v_stride, int dtype, void* k_codes,
                                void* v_codes, void* words, int num_pages, int page_size, int g, int dim, const int32_t* positions,
                                const int32_t* req_of_token, const int32_t* block_table, int table_width, int n_tokens, int vector,
                                int32_t* error, cudaStream_t stream) {
  if (dim < 8 || dim > 256 || dim % 8 || page_size < 1 || g < 1) return YALIS_ERR_SHAPE;
  if (n_tokens <= 0) return YALIS_OK;
  YALIS_DISPATCH_DTYPE(dtype, T, {
    RowParams<T> p = {};
    p.k = static_cast<const T*>(k); p.v = static_cast<const T*>(v);
    p.k_out = static_cast<T*>(k); p.v_out = static_cast<T*>(v);
    p.k_stride = k_stride; p.v_stride = v_stride;
    p.positions = positions; p.req_of_token = req_of_token; p.block_table = block_table;
    p.table_width = table_width; p.n_tokens = n_tokens; p.vector = vector; p.error = error;
    p.pages = packed_pages(k_codes, v_codes, words, num_pages, page_size, g, dim);
    return write ? launch_rows<T, true>(p, n_tokens, stream) : launch_rows<T, false>(p, n_tokens, stream);
  });
}

YALIS_API int yalis_packed_unpack(void* k_codes, void* v_codes, void* words, int num_pages, int page_size, int g, int dim, const int32_t* positions,
                                  const int32_t* q_start, const int32_t* block_table, int table_width, int n_requests, int width, int window,
                                  int skip_single, void* k_out, void* v_out, void* marks, int32_t* some_marked, int marked_by,
                                  int32_t* table_out, int32_t* zeroed, int n_zeroed, int32_t* error, cudaStream_t stream) {
  if ((dim != 64 && dim != 128) || page_size < 1 || g < 1 || width < 1) return YALIS_ERR_SHAPE;
  if (n_requests <= 0) return YALIS_OK;
  UnpackParams p = {};
  p.n_zeroed = n_zeroed;
  p.k_out = static_cast<__nv_bfloat16*>(k_out); p.v_out = static_cast<__nv_bfloat16*>(v_out); p.marks = static_cast<uint32_t*>(marks);
  p.some_marked = some_marked; p.marked_by = marked_by; p.table_out = table_out; p.zeroed = zeroed;
  p.positions = positions; p.q_start = q_start; p.block_table = block_table; p.table_width = table_width; p.n_requests = n_requests;
  p.width = width; p.window = window; p.skip_single = skip_single; p.error = error;
  p.pages = packed_pages(k_codes, v_codes, words, num_pages, page_size, g, dim);
  const long long most = (long long)width * g * n_requests, resident = 4LL * yalis_sm_count();
  return yalis_launch(packed_unpack_kernel, dim3((unsigned)(most < resident ? most : resident)), dim3(kUnpackThreads), 0, stream, p);
}

YALIS_SLOTS(yalis_packed_rows)
YALIS_SLOTS(yalis_packed_unpack)
