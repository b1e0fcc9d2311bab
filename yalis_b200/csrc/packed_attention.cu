// Attention over pages held in 4 bits (packed.cuh), and the sums of the weights that every cached token receives.
//
// With q a query of one head, c_j, z_j, s_j the codes, zero and step of key j and d_j, y_j, t_j those of its value:
//   S_j = scale * s_j * (q . c_j - z_j sum(q)),   P = softmax of S over the keys seen,   O = sum_j (P_j t_j) (d_j - y_j)
// and, where sums are kept, A_j += P_j for every query row and head of j's KV head.  A row that sees nothing gives zeros.
//
// The general form: a block per (token, head), a thread per key of a tile for the scores and per element for O; scores, weights
// and sums in float32.  It takes every size; its weights' normaliser, log2(sum exp S), goes to memory for the sums, which a second
// kernel adds key by key in the order of the rows.
#include "packed.cuh"
#include "slots.cuh"

namespace {

constexpr int kThreads = 128;

struct AttentionParams {
  const void* q;               // [N, q_stride]
  long long q_stride;
  void* out;                   // [N, out_stride]
  long long out_stride;
  const int32_t* positions;    // [N] the last place of the cache that a row sees
  const int32_t* q_start;      // [R + 1]
  const int32_t* block_table;  // [R, table_width]
  int table_width, n_requests, n_tokens, nh, per, window;
  int reach;                   // places that the table has
  float scale;
  float* lse2;                 // [N, nh] the logarithm to base two of a row's sum of exponentials, or null
  float* sums;                 // [pages, g, page_size] or null
  int32_t* error;
  PackedPages pages;
};

// The request of a token (the last whose range starts at or before it), -1 for rows of no request.
__device__ __forceinline__ int request_of(const AttentionParams& p, int token) {
  if (token < p.q_start[0] || token >= p.q_start[p.n_requests]) return -1;
  int lo = 0, hi = p.n_requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.q_start[mid] <= token) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// q . c of one row, and the score from it.
__device__ __forceinline__ float code_product(const uint32_t* row, const float* q, int words) {
  float acc = 0.f;
  for (int w = 0; w < words; ++w) {
    const uint32_t c = row[w];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = fmaf((float)((c >> (4 * i)) & 15u), q[8 * w + i], acc);
  }
  return acc;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) packed_attention_general_kernel(const AttentionParams p) {
  __shared__ float q[256], weight[kThreads], zero[kThreads], scratch[32];
  __shared__ long long row_at[kThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int token = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, dim = p.pages.dim, words = dim / 8, kvh = head / p.per;
  const int req = request_of(p, token);
  if (req < 0) return;
  const T* src = static_cast<const T*>(p.q) + (long long)token * p.q_stride + (long long)head * dim;
  float part = 0.f;
  for (int i = tid; i < dim; i += kThreads) part += q[i] = to_f32<T>(src[i]);
  const float q_sum = block_sum(part, scratch);
  const int place = p.positions[token], first = p.window > 0 ? max(0, place - p.window + 1) : 0, last = min(place, p.reach - 1);
  if (place > last && tid == 0 && p.error) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);       // (places behind the table have no page)
  const int32_t* table_row = p.block_table + (size_t)req * p.table_width;
  float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
  for (long long j0 = first; j0 <= last; j0 += kThreads) {
    const int j = (int)(j0 + tid), n = (int)min((long long)kThreads, last - j0 + 1);
    float score = -INFINITY, step = 0.f, z = 0.f;
    long long at = -1;
    if (tid < n) {
      int row;
      const int page = page_of(p.pages, table_row, p.table_width, j, row);
      if (page < 0) {
        if (p.error) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);
      } else {
        at = (long long)row_index(p.pages, page, kvh, row);
        const uint32_t word = p.pages.words[at];
        score = p.scale * step_of(word & 0xFFFFu) * fmaf(-zero_of(word), q_sum, code_product(p.pages.k + at * words, q, words));
        step = step_of(word >> 16);
        z = zero_of(word >> 16);
      }
    }
    const float m_new = fmaxf(m, block_max(score, scratch));
    const float keep = m_new == -INFINITY ? 1.f : expf(m - m_new);
    const float e = at < 0 ? 0.f : expf(score - m_new);
    l = l * keep + block_sum(e, scratch);
    __syncthreads();
    weight[tid] = at < 0 ? 0.f : e * step;
    zero[tid] = z;
    row_at[tid] = at;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int d = tid + h * kThreads;
      if (d < dim) {
        acc[h] *= keep;
        for (int i = 0; i < n; ++i) {
          if (row_at[i] < 0) continue;
          const uint32_t c = (p.pages.v[row_at[i] * words + (d >> 3)] >> (4 * (d & 7))) & 15u;
          acc[h] = fmaf(weight[i], (float)c - zero[i], acc[h]);
        }
      }
    }
    m = m_new;
  }
  T* dst = static_cast<T*>(p.out) + (long long)token * p.out_stride + (long long)head * dim;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int d = tid + h * kThreads;
    if (d < dim) dst[d] = from_f32<T>(l == 0.f ? 0.f : acc[h] / l);
  }
  if (tid == 0 && p.lse2) p.lse2[(size_t)token * p.nh + head] = (m + logf(l)) * 1.4426950408889634f;
}

// A block per (tile of keys, KV head, request), a thread per key: the rows that see the key, in their order.
template <typename T>
__global__ void __launch_bounds__(kThreads) packed_weight_sums_general_kernel(const AttentionParams p) {
  __shared__ float q[256], scratch[32];
  pdl_launch_dependents();
  pdl_wait();
  const int j0 = blockIdx.x * kThreads, j = j0 + threadIdx.x, kvh = blockIdx.y, req = blockIdx.z, dim = p.pages.dim, words = dim / 8;
  const int t0 = p.q_start[req], t1 = p.q_start[req + 1];
  if (t0 >= t1) return;
  const int32_t* table_row = p.block_table + (size_t)req * p.table_width;
  int row;
  const int page = page_of(p.pages, table_row, p.table_width, j, row);
  const size_t at = page < 0 ? 0 : row_index(p.pages, page, kvh, row);
  const uint32_t word = page < 0 ? 0u : p.pages.words[at];
  float total = 0.f;
  bool seen = false;
  for (int t = t0; t < t1; ++t) {
    const int last = p.positions[t], first = p.window > 0 ? max(0, last - p.window + 1) : 0;
    if (last < j0 || first > j0 + kThreads - 1) continue;
    const bool sees = page >= 0 && j <= last && j >= first;
    for (int h = 0; h < p.per; ++h) {
      const int head = kvh * p.per + h;
      const T* src = static_cast<const T*>(p.q) + (long long)t * p.q_stride + (long long)head * dim;
      __syncthreads();
      float part = 0.f;
      for (int i = threadIdx.x; i < dim; i += kThreads) part += q[i] = to_f32<T>(src[i]);
      const float q_sum = block_sum(part, scratch);
      if (sees) {
        const float s = p.scale * step_of(word & 0xFFFFu) * fmaf(-zero_of(word), q_sum, code_product(p.pages.k + at * words, q, words));
        total += exp2f(s * 1.4426950408889634f - p.lse2[(size_t)t * p.nh + head]);
        seen = true;
      }
    }
  }
  if (seen) atomicAdd(p.sums + at, total);       // (one addition a token and KV head, whatever the number of rows)
}

}  // namespace

namespace {

bool params_of(AttentionParams& p, const void* q, long long q_stride, void* k_codes, void* v_codes, void* words, int num_pages, int page_size,
               int g, int dim, const int32_t* positions, const int32_t* q_start, const int32_t* block_table, int table_width, int n_requests,
               int nh, float scale, int window) {
  if (dim < 8 || dim > 256 || dim % 8 || page_size < 1 || g < 1 || nh % g || nh > 65535 || n_requests > 65535) return false;
  p = {};
  p.q = q; p.q_stride = q_stride;
  p.positions = positions; p.q_start = q_start; p.block_table = block_table; p.table_width = table_width;
  p.n_requests = n_requests; p.nh = nh; p.per = nh / g; p.window = window; p.scale = scale;
  p.reach = (int)min((long long)table_width * page_size, 0x7fffffffll);
  p.pages = packed_pages(k_codes, v_codes, words, num_pages, page_size, g, dim);
  return true;
}

}  // namespace

YALIS_API int yalis_packed_attention_general(const void* q, long long q_stride, int dtype, void* out, long long out_stride, void* k_codes,
                                             void* v_codes, void* words, int num_pages, int page_size, int g, int dim,
                                             const int32_t* positions, const int32_t* q_start, const int32_t* block_table, int table_width,
                                             int n_requests, int n_tokens, int nh, float scale, int window, float* lse2, int32_t* error,
                                             cudaStream_t stream) {
  AttentionParams p;
  if (!params_of(p, q, q_stride, k_codes, v_codes, words, num_pages, page_size, g, dim, positions, q_start, block_table, table_width, n_requests,
                 nh, scale, window))
    return YALIS_ERR_SHAPE;
  if (n_tokens <= 0 || n_requests <= 0) return YALIS_OK;
  p.out = out; p.out_stride = out_stride; p.n_tokens = n_tokens; p.lse2 = lse2; p.error = error;
  YALIS_DISPATCH_DTYPE(dtype, T, return yalis_launch(packed_attention_general_kernel<T>, dim3(n_tokens, nh), dim3(kThreads), 0, stream, p));
}

// Adds to `sums` the weights that the step's rows give the cached tokens; `lse2` [N, nh] from the attention of the same step.
YALIS_API int yalis_packed_weight_sums_general(const void* q, long long q_stride, int dtype, void* k_codes, void* v_codes, void* words,
                                               int num_pages, int page_size, int g, int dim, const int32_t* positions, const int32_t* q_start,
                                               const int32_t* block_table, int table_width, int n_requests, int max_kv_len, int nh, float scale,
                                               int window, float* lse2, float* sums, cudaStream_t stream) {
  AttentionParams p;
  if (!params_of(p, q, q_stride, k_codes, v_codes, words, num_pages, page_size, g, dim, positions, q_start, block_table, table_width, n_requests,
                 nh, scale, window) || g > 65535)
    return YALIS_ERR_SHAPE;
  if (n_requests <= 0 || max_kv_len <= 0) return YALIS_OK;
  p.lse2 = lse2; p.sums = sums;
  YALIS_DISPATCH_DTYPE(dtype, T, return yalis_launch(packed_weight_sums_general_kernel<T>, dim3((unsigned)((max_kv_len + kThreads - 1LL) / kThreads), g,
                                                                                                  n_requests), dim3(kThreads), 0, stream, p));
}

YALIS_SLOTS(yalis_packed_attention_general)
YALIS_SLOTS(yalis_packed_weight_sums_general)
