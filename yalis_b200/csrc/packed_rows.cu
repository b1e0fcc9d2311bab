// Rows of keys and values into pages held in 4 bits, and back.
//
// A row of one token and KV head is taken by dim / 8 neighbouring lanes (a group of 4, 8, 16 or 32), eight values a lane: the
// row's extremes by shuffles, then every lane its word of eight codes.  Keys and values are rows of one grid.
// Bound by memory: 2 dim values read and dim + 4 bytes written a token and KV head (bfloat16: 512 -> 132 B at 128).
#include "packed.cuh"

namespace {

constexpr int kThreads = 128;

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
  int vector;                  // 1: rows start on boundaries of eight values
  int32_t* error;
  PackedPages pages;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vector, float (&x)[8]) {
  if (vector) {
    const float4 a = load4_f32(p), b = load4_f32(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(p[i]);
  }
}

// What a group of lanes works on: row `index` of the grid is token index / (2 g), KV head and key or value from the rest.
struct Place {
  int token, kvh, is_v;
  bool real;                   // a token with a page
  size_t row;
};

template <typename T>
__device__ __forceinline__ Place place_of(const RowParams<T>& p, long long index, int lane_in_row) {
  Place o;
  const int per_token = 2 * p.pages.g;
  o.token = (int)(index / per_token);
  const int rest = (int)(index - (long long)o.token * per_token);
  o.is_v = rest & 1;
  o.kvh = rest >> 1;
  o.real = o.token < p.n_tokens;
  o.row = 0;
  if (o.real) {
    const int req = p.req_of_token[o.token], at = p.positions[o.token];
    o.real = req >= 0 && at >= 0;
    if (o.real) {
      int row;
      const int page = page_of(p.pages, p.block_table + (size_t)req * p.table_width, p.table_width, at, row);
      if (page < 0) {
        o.real = false;
        if (lane_in_row == 0 && p.error) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);
      } else {
        o.row = row_index(p.pages, page, o.kvh, row);
      }
    }
  }
  return o;
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) packed_rows_write_kernel(const RowParams<T> p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & (LANES - 1);
  const long long index = ((long long)blockIdx.x * kThreads + threadIdx.x) / LANES;
  const Place at = place_of(p, index, lane);
  const bool mine = at.real && lane * 8 < p.pages.dim;
  float x[8];
  if (mine) {
    const T* src = at.is_v ? p.v + (long long)at.token * p.v_stride : p.k + (long long)at.token * p.k_stride;
    load8<T>(src + (size_t)at.kvh * p.pages.dim + lane * 8, p.vector, x);
  }
  float lo = 0.f, hi = 0.f;
  int odd = 0;
  if (mine) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      odd |= !(fabsf(x[i]) <= kPackedLargest);
    }
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    odd |= __shfl_xor_sync(0xffffffffu, odd, o);
  }
  if (!mine) return;
  uint32_t codes = 0, word = 0x7FC0u;                          // not a number: all codes 0
  if (!odd) {
    const float step = step_for(lo, hi), first = multiple_of(lo, step);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = (int)fminf(multiple_of(x[i], step) - first, 15.f);
      codes |= (uint32_t)max(c, 0) << (4 * i);
    }
    word = (__float_as_uint(step) >> 16) | (uint32_t)(int)-first;
  }
  (at.is_v ? p.pages.v : p.pages.k)[at.row * (p.pages.dim / 8) + lane] = codes;
  if (lane == 0) reinterpret_cast<uint16_t*>(p.pages.words + at.row)[at.is_v] = (uint16_t)word;
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) packed_rows_read_kernel(const RowParams<T> p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & (LANES - 1);
  const long long index = ((long long)blockIdx.x * kThreads + threadIdx.x) / LANES;
  const Place at = place_of(p, index, lane);
  if (at.token >= p.n_tokens || lane * 8 >= p.pages.dim) return;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};       // a token without a page reads as zeros
  if (at.real) {
    const uint32_t codes = (at.is_v ? p.pages.v : p.pages.k)[at.row * (p.pages.dim / 8) + lane];
    const uint32_t word = reinterpret_cast<const uint16_t*>(p.pages.words + at.row)[at.is_v];
    const float step = step_of(word), zero = zero_of(word);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ((float)((codes >> (4 * i)) & 15u) - zero) * step;
  }
  T* dst = (at.is_v ? p.v_out : p.k_out) + ((size_t)at.token * p.pages.g + at.kvh) * p.pages.dim + lane * 8;
  store4(dst, make_float4(x[0], x[1], x[2], x[3]));
  store4(dst + 4, make_float4(x[4], x[5], x[6], x[7]));
}

template <typename T, bool WRITE>
int launch_rows(const RowParams<T>& p, cudaStream_t stream) {
  const int lanes = p.pages.dim <= 32 ? 4 : p.pages.dim <= 64 ? 8 : p.pages.dim <= 128 ? 16 : 32;
  const long long rows = (long long)p.n_tokens * p.pages.g * 2, per_block = kThreads / lanes, blocks = (rows + per_block - 1) / per_block;
  if (blocks > 0x7fffffffll) return YALIS_ERR_SHAPE;
  const dim3 grid((unsigned)blocks), block(kThreads);
#define YALIS_ROWS(L) \
  yalis_launch(WRITE ? packed_rows_write_kernel<T, L> : packed_rows_read_kernel<T, L>, grid, block, 0, stream, p)
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
// and the counters of the kernels behind it at zero.  Exact: every value is a bfloat16 number.  A block takes a page of one KV
// head, a thread eight codes at a time.  Bound by the writes (512 B a token and KV head at 128), most of which the reader finds
// in the L2.
constexpr int kUnpackPage = 64;

struct UnpackParams {
  __nv_bfloat16* k_out;        // [R * width, g, kUnpackPage, dim]
  __nv_bfloat16* v_out;
  int32_t* table_out;          // [R, width]
  int32_t* zeroed;             // [n_zeroed] counters (no more than the launch has threads)
  long long n_zeroed;
  const int32_t* positions;
  const int32_t* q_start;      // [R + 1]
  const int32_t* block_table;
  int table_width, width, window, skip_single;
  int32_t* error;
  PackedPages pages;
};

__global__ void __launch_bounds__(256) packed_unpack_kernel(const UnpackParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int index = blockIdx.x, kvh = blockIdx.y, req = blockIdx.z, words = p.pages.dim / 8;
  if (threadIdx.x == 0) {
    if (kvh == 0) p.table_out[(size_t)req * p.width + index] = req * p.width + index;
  }
  const long long thread = (((long long)req * p.pages.g + kvh) * p.width + index) * 256 + threadIdx.x;
  if (thread < p.n_zeroed) p.zeroed[thread] = 0;
  const int t0 = p.q_start[req], n = p.q_start[req + 1] - t0;
  if (n <= 0 || (p.skip_single && n == 1)) return;
  const int last = p.positions[t0 + n - 1], begin = p.positions[t0], key0 = index * kUnpackPage;
  const int first = p.window > 0 ? max(0, begin - p.window + 1) : 0;
  if (key0 > last || key0 + kUnpackPage <= first) return;
  const size_t to = (((size_t)req * p.width + index) * p.pages.g + kvh) * kUnpackPage;
  const int rows = min(kUnpackPage, last - key0 + 1);
  for (int i = threadIdx.x; i < rows * words; i += 256) {
    const int r = i / words, w = i - r * words, key = key0 + r;
    int row;
    const int page = page_of(p.pages, p.block_table + (size_t)req * p.table_width, p.table_width, key, row);
    uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
    if (page >= 0) {
      const size_t at = row_index(p.pages, page, kvh, row);
      const uint32_t word = p.pages.words[at], kc = p.pages.k[at * words + w], vc = p.pages.v[at * words + w];
      const float ks = step_of(word & 0xFFFFu), kz = zero_of(word), vs = step_of(word >> 16), vz = zero_of(word >> 16);
      uint32_t* out[2] = {&k.x, &v.x};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(((float)(kc >> (8 * e) & 15u) - kz) * ks, ((float)(kc >> (8 * e + 4) & 15u) - kz) * ks);
        const __nv_bfloat162 b = __floats2bfloat162_rn(((float)(vc >> (8 * e) & 15u) - vz) * vs, ((float)(vc >> (8 * e + 4) & 15u) - vz) * vs);
        out[0][e] = *reinterpret_cast<const uint32_t*>(&a);
        out[1][e] = *reinterpret_cast<const uint32_t*>(&b);
      }
    } else if (key >= first && w == 0 && p.error) {
      atomicOr(p.error, YALIS_FLAG_BAD_PAGE);
    }
    reinterpret_cast<uint4*>(p.k_out)[(to + r) * words + w] = k;
    reinterpret_cast<uint4*>(p.v_out)[(to + r) * words + w] = v;
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
    p.pages = {static_cast<uint32_t*>(k_codes), static_cast<uint32_t*>(v_codes), static_cast<uint32_t*>(words), num_pages, page_size, g, dim};
    return write ? launch_rows<T, true>(p, stream) : launch_rows<T, false>(p, stream);
  });
}

YALIS_API int yalis_packed_unpack(void* k_codes, void* v_codes, void* words, int num_pages, int page_size, int g, int dim, const int32_t* positions,
                                  const int32_t* q_start, const int32_t* block_table, int table_width, int n_requests, int width, int window,
                                  int skip_single, void* k_out, void* v_out, int32_t* table_out, int32_t* zeroed, int n_zeroed, int32_t* error,
                                  cudaStream_t stream) {
  if (dim < 8 || dim > 256 || dim % 8 || page_size < 1 || g < 1 || g > 65535 || n_requests > 65535 || width < 1) return YALIS_ERR_SHAPE;
  if (n_requests <= 0) return YALIS_OK;
  if (n_zeroed > (long long)width * g * n_requests * 256) return YALIS_ERR_SHAPE;
  UnpackParams p = {};
  p.n_zeroed = n_zeroed;
  p.k_out = static_cast<__nv_bfloat16*>(k_out); p.v_out = static_cast<__nv_bfloat16*>(v_out); p.table_out = table_out; p.zeroed = zeroed;
  p.positions = positions; p.q_start = q_start; p.block_table = block_table; p.table_width = table_width; p.width = width;
  p.window = window; p.skip_single = skip_single; p.error = error;
  p.pages = {static_cast<uint32_t*>(k_codes), static_cast<uint32_t*>(v_codes), static_cast<uint32_t*>(words), num_pages, page_size, g, dim};
  return yalis_launch(packed_unpack_kernel, dim3(width, g, n_requests), dim3(256), 0, stream, p);
}
