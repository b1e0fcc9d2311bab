// Sums of attention weights per cached token over pages held in 4 bits (packed.cuh), on the tensor cores (head sizes 64 and 128).
//
// A_j += sum over the step's rows n that see key j, and over the heads of j's KV head, of exp(S_nj - lse_n), with S as in
// packed_attention.cu and lse_n, the logarithm of row n's sum of exponentials, from the attention before.  A block owns keys, so that
// every token's sum is one addition to memory, whatever the number of rows, and its order fixed: a warp keeps 32 keys' codes less
// their zeros as bfloat16 operands in registers and walks the rows (columns of the product, see packed_attention_mma.cu) that see
// any of the block's keys.  The rows' queries lie in shared memory in the operand's order, COLUMNS at a time, written from registers
// that were loaded a round before.  Two groups of four warps have 32 keys each; the four divide the columns among them and add up at the
// end.
//
// Steps of few rows (single tokens) leave their scores in memory while the attention computes them: a second kernel raises and adds them,
// a thread per key.  That moves 8 bytes a row and key, where taking the products once more reads the keys' codes again (16 requests of
// 2,100 to 4,000 tokens, 32 heads of 128 over 8: 58 us by products, 8.5 by scores).
#include "packed.cuh"
#include "slots.cuh"

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kKeys = 32;      // keys of a warp

struct SumsParams {
  const void* q;               // [N, q_stride]
  long long q_stride;
  const int32_t* positions;    // [N]
  const int32_t* q_start;      // [R + 1]
  const int32_t* block_table;
  int table_width, nh, per, window, q_vector;
  int only_single;             // 1: requests that bring more than one token are left to another kernel
  float scale_log2;
  const float* lse2;           // [N, nh] in powers of two
  float* sums;                 // [pages, g, page_size]
  PackedPages pages;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Codes i and i + 4 of the eight in w, less the row's zero (16 + zero twice in z), as a bfloat16 pair.
template <int I>
__device__ __forceinline__ uint32_t signed_pair(uint32_t w, uint32_t sixteens, uint32_t z) {
  const uint32_t at = I == 0 ? w << 3 : w >> (I == 0 ? 0 : 4 * I - 3);
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00780078, %2, 0xEA;" : "=r"(r) : "r"(at), "r"(sixteens));
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&r), *reinterpret_cast<const __nv_bfloat162*>(&z));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// KG groups of 32 keys by CG groups of columns a block; COLUMNS of queries in shared memory at a time.
template <typename T, int DIM, int PARTS, int KG, int CG, int COLUMNS>
__global__ void __launch_bounds__(kThreads, 1) packed_weight_sums_kernel(const SumsParams p) {
  constexpr int W = DIM / 32;                  // words of a K row that a lane takes
  constexpr int PIECES = COLUMNS * DIM / 8;    // of eight elements
  constexpr int OWN = (PIECES + kThreads - 1) / kThreads;
  static_assert(KG * CG == kWarps, "a warp has a group of keys and a group of columns");
  __shared__ uint4 q_s[PARTS][COLUMNS / 8 * W * 32];
  __shared__ float lse_s[COLUMNS];
  __shared__ int last_s[COLUMNS];
  __shared__ float sum_s[CG > 1 ? CG : 1][CG > 1 ? KG * kKeys : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.x % p.pages.g, req = blockIdx.y, kg = warp / CG, cg = warp % CG;
  const int block0 = blockIdx.x / p.pages.g * (KG * kKeys), key0 = block0 + kg * kKeys;
  pdl_launch_dependents();
  pdl_wait();
  const int tok0 = p.q_start[req], n = p.q_start[req + 1] - tok0;
  if (n <= 0 || (p.only_single && n > 1)) return;
  const int begin = p.positions[tok0], last = p.positions[tok0 + n - 1];
  if (block0 > last || last < 0) return;
  // Rows stand at consecutive places: those that see a key of the block are [t_lo, t_hi).
  const int t_lo = min(max(block0 - begin, 0), n);
  const int t_hi = p.window > 0 ? (int)min((long long)n, max(0ll, (long long)block0 + KG * kKeys - 1 + p.window - begin)) : n;
  if (t_lo >= t_hi) return;
  const int first = p.window > 0 ? max(0, begin - p.window + 1) : 0;      // the first key that any row sees

  // ---- this warp's keys: rows g, g + 8, g + 16, g + 24 of a lane ----
  uint32_t sixteens;
  asm volatile("mov.b32 %0, 0x41804180;" : "=r"(sixteens));
  const int32_t* table_row = p.block_table + (size_t)req * p.table_width;
  uint32_t kf[2][2 * W][4];
  float step[2][2];
  size_t at[2][2];
  bool there[2][2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t words[2][W], z[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int key = key0 + half * 16 + e * 8 + g;
      int row, page = -1;
      if (key <= last && key >= first) page = page_of(p.pages, table_row, p.table_width, key, row);
      there[half][e] = page >= 0;
      at[half][e] = page >= 0 ? row_index(p.pages, page, kvh, row) : 0;
      uint32_t word = 0u;
#pragma unroll
      for (int w = 0; w < W; ++w) words[e][w] = 0u;
      if (page >= 0) {
        word = p.pages.words[at[half][e]];
        const uint32_t* src = p.pages.k + at[half][e] * (DIM / 8) + t * W;
        if constexpr (W == 4) *reinterpret_cast<uint4*>(words[e]) = *reinterpret_cast<const uint4*>(src);
        else *reinterpret_cast<uint2*>(words[e]) = *reinterpret_cast<const uint2*>(src);
      }
      step[half][e] = step_of(word & 0xFFFFu) * p.scale_log2;
      z[e] = ((word & 15u) << 3 | 0x4180u) * 0x10001u;
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        kf[half][2 * w][e] = signed_pair<0>(words[e][w], sixteens, z[e]);
        kf[half][2 * w][2 + e] = signed_pair<1>(words[e][w], sixteens, z[e]);
        kf[half][2 * w + 1][e] = signed_pair<2>(words[e][w], sixteens, z[e]);
        kf[half][2 * w + 1][2 + e] = signed_pair<3>(words[e][w], sixteens, z[e]);
      }
    }
  }

  // ---- the columns, a round of COLUMNS at a time ----
  const int c_lo = t_lo * p.per, c_hi = t_hi * p.per;
  auto load = [&](int c0, float (&x)[OWN][8]) {
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int piece = i * kThreads + threadIdx.x, column = c0 + piece / (DIM / 8);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[i][k] = 0.f;
      if (piece < PIECES && column < c_hi) {
        const T* src = static_cast<const T*>(p.q) + (long long)(tok0 + column / p.per) * p.q_stride +
                       (long long)(kvh * p.per + column % p.per) * DIM + piece % (DIM / 8) * 8;
        if (p.q_vector) {
          const float4 a = load4_f32(src), b = load4_f32(src + 4);
          x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w;
          x[i][4] = b.x; x[i][5] = b.y; x[i][6] = b.z; x[i][7] = b.w;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[i][k] = to_f32<T>(src[k]);
        }
      }
    }
  };
  float x[OWN][8], total[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
  load(c_lo, x);
  for (int c0 = c_lo; c0 < c_hi; c0 += COLUMNS) {
    if (c0 > c_lo) __syncthreads();              // the round before has been read
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int piece = i * kThreads + threadIdx.x;
      if (piece < PIECES) {
        const int column = piece / (DIM / 8), k = piece % (DIM / 8);
        const int to = ((column >> 3) * W + k % W) * 32 + (column & 7) * 4 + k / W;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          uint32_t pair[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(x[i][j], x[i][j + 4]);
            pair[j] = *reinterpret_cast<const uint32_t*>(&v);
            x[i][j] -= __uint_as_float(pair[j] << 16);
            x[i][j + 4] -= __uint_as_float(pair[j] & 0xFFFF0000u);
          }
          q_s[part][to] = make_uint4(pair[0], pair[1], pair[2], pair[3]);
        }
      }
    }
    for (int c = threadIdx.x; c < COLUMNS; c += kThreads) {
      const int column = c0 + c;
      const bool real = column < c_hi;
      lse_s[c] = real ? p.lse2[(size_t)(tok0 + column / p.per) * p.nh + kvh * p.per + column % p.per] : INFINITY;
      last_s[c] = real ? p.positions[tok0 + column / p.per] : -1;
    }
    __syncthreads();
    if (c0 + COLUMNS < c_hi) load(c0 + COLUMNS, x);
    const int blocks = min(COLUMNS, c_hi - c0 + 7) / 8;
    // Whether every column of the round sees every key of the warp (positions ascend).
    const int low = begin + c0 / p.per, high = begin + (min(c0 + COLUMNS, c_hi) - 1) / p.per;
    const bool masked = c0 + COLUMNS > c_hi || low < key0 + kKeys - 1 || (p.window > 0 && high - p.window + 1 > key0);
    for (int nb = cg; nb < blocks; nb += CG) {
      float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int part = PARTS - 1; part >= 0; --part) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint4 b = q_s[part][(nb * W + w) * 32 + lane];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            mma_bf16(acc[half], kf[half][2 * w], b.x, b.y);
            mma_bf16(acc[half], kf[half][2 * w + 1], b.z, b.w);
          }
        }
      }
      const float2 lse = *reinterpret_cast<const float2*>(lse_s + nb * 8 + 2 * t);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float a = fmaf(step[half][e], acc[half][2 * e], -lse.x), b = fmaf(step[half][e], acc[half][2 * e + 1], -lse.y);
          float pa = PARTS == 1 ? exp2_fast(a) : exp2f(a), pb = PARTS == 1 ? exp2_fast(b) : exp2f(b);
          if (masked) {
            const int2 sees = *reinterpret_cast<const int2*>(last_s + nb * 8 + 2 * t);
            const int key = key0 + half * 16 + e * 8 + g;
            if (key > sees.x || (p.window > 0 && key <= sees.x - p.window)) pa = 0.f;
            if (key > sees.y || (p.window > 0 && key <= sees.y - p.window)) pb = 0.f;
          }
          total[half][e] += pa + pb;
        }
      }
    }
  }
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      total[half][e] += __shfl_xor_sync(0xffffffffu, total[half][e], 1);
      total[half][e] += __shfl_xor_sync(0xffffffffu, total[half][e], 2);
    }
  if constexpr (CG > 1) {
    if (t == 0)
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 2; ++e) sum_s[cg][kg * kKeys + half * 16 + e * 8 + g] = total[half][e];
    __syncthreads();
    if (cg != 0) return;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        total[half][e] = 0.f;
#pragma unroll
        for (int i = 0; i < CG; ++i) total[half][e] += sum_s[i][kg * kKeys + half * 16 + e * 8 + g];
      }
  }
  if (t == 0)
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (there[half][e]) atomicAdd(p.sums + at[half][e], total[half][e]);
}

template <typename T, int DIM, int PARTS>
int launch_sums(const SumsParams& p, int n_requests, int max_kv_len, cudaStream_t stream) {
  const long long blocks = (max_kv_len + 2LL * kKeys - 1) / (2 * kKeys) * p.pages.g;
  if (n_requests > 65535 || blocks > 0x7fffffff) return YALIS_ERR_SHAPE;
  const dim3 grid((unsigned)blocks, n_requests);
  return yalis_launch(packed_weight_sums_kernel<T, DIM, PARTS, 2, 4, 64 / (PARTS == 1 ? 1 : 2)>, grid, dim3(kThreads), 0, stream, p);
}

// From scores: a thread per key of a KV head, over the rows that see it in their order.  SINGLE: only of requests that bring one token, with a
// row of scores a request.
template <bool SINGLE>
__global__ void __launch_bounds__(256) packed_sums_of_scores_kernel(const SumsParams p, const float* scores, long long stride) {
  pdl_launch_dependents();
  pdl_wait();
  const int key = blockIdx.x * 256 + threadIdx.x, kvh = blockIdx.y, req = blockIdx.z;
  const int tok0 = p.q_start[req], n = p.q_start[req + 1] - tok0;
  if (n <= 0 || (SINGLE && n > 1)) return;
  const int last = p.positions[tok0 + n - 1], begin = p.positions[tok0];
  if (key >= stride || key > last || (p.window > 0 && key <= begin - p.window)) return;
  int in_page;
  const int page = page_of(p.pages, p.block_table + (size_t)req * p.table_width, p.table_width, key, in_page);
  if (page < 0) return;
  if constexpr (SINGLE) scores += ((long long)req - tok0) * p.nh * stride;
  float total = 0.f;
  for (int t = 0; t < n; ++t) {
    const int place = p.positions[tok0 + t];
    if (key > place || (p.window > 0 && key <= place - p.window)) continue;
    const size_t first = (size_t)(tok0 + t) * p.nh + kvh * p.per;
    for (int h = 0; h < p.per; h += 4) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = h + i < p.per ? scores[(first + h + i) * stride + key] - p.lse2[first + h + i] : -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) total += exp2f(x[i]);
    }
  }
  atomicAdd(p.sums + row_index(p.pages, page, kvh, in_page), total);
}

}  // namespace

namespace {

SumsParams params_of(const void* q, long long q_stride, int num_pages, int page_size, int g, int dim, const int32_t* positions,
                     const int32_t* q_start, const int32_t* block_table, int table_width, int nh, float scale, int window, int only_single,
                     float* lse2, float* sums) {
  SumsParams p = {};
  p.q = q; p.q_stride = q_stride; p.positions = positions; p.q_start = q_start; p.block_table = block_table; p.table_width = table_width;
  p.nh = nh; p.per = nh / g; p.window = window; p.only_single = only_single; p.scale_log2 = scale * 1.4426950408889634f;
  p.lse2 = lse2; p.sums = sums;
  p.pages = packed_pages(nullptr, nullptr, nullptr, num_pages, page_size, g, dim);
  return p;
}

}  // namespace

YALIS_API int yalis_packed_weight_sums(const void* q, long long q_stride, int dtype, void* k_codes, void* v_codes, void* words, int num_pages,
                                       int page_size, int g, int dim, const int32_t* positions, const int32_t* q_start,
                                       const int32_t* block_table, int table_width, int n_requests, int max_kv_len, int nh, float scale,
                                       int window, int q_vector, int only_single, float* lse2, float* sums, cudaStream_t stream) {
  if ((dim != 64 && dim != 128) || g < 1 || nh % g || page_size < 1) return YALIS_ERR_SHAPE;
  if (n_requests <= 0 || max_kv_len <= 0) return YALIS_OK;
  SumsParams p = params_of(q, q_stride, num_pages, page_size, g, dim, positions, q_start, block_table, table_width, nh, scale, window, only_single,
                           lse2, sums);
  p.q_vector = q_vector;
  p.pages.k = static_cast<uint32_t*>(k_codes); p.pages.v = static_cast<uint32_t*>(v_codes); p.pages.words = static_cast<uint32_t*>(words);
  if (dtype == YALIS_BF16)
    return dim == 64 ? launch_sums<__nv_bfloat16, 64, 1>(p, n_requests, max_kv_len, stream)
                     : launch_sums<__nv_bfloat16, 128, 1>(p, n_requests, max_kv_len, stream);
  if (dtype == YALIS_F32)
    return dim == 64 ? launch_sums<float, 64, 3>(p, n_requests, max_kv_len, stream) : launch_sums<float, 128, 3>(p, n_requests, max_kv_len, stream);
  return YALIS_ERR_DTYPE;
}

// The same from scores [N, nh, score_stride] ([R, nh, score_stride] of single tokens beside others) that the attention of the step left
// (yalis_packed_attention_mma).
YALIS_API int yalis_packed_sums_of_scores(float* scores, long long score_stride, int num_pages, int page_size, int g, int dim,
                                          const int32_t* positions, const int32_t* q_start, const int32_t* block_table, int table_width,
                                          int n_requests, int max_kv_len, int nh, int window, int only_single, float* lse2, float* sums,
                                          cudaStream_t stream) {
  if (g < 1 || g > 65535 || nh % g || page_size < 1 || n_requests > 65535) return YALIS_ERR_SHAPE;
  if (n_requests <= 0 || max_kv_len <= 0) return YALIS_OK;
  const SumsParams p = params_of(nullptr, 0, num_pages, page_size, g, dim, positions, q_start, block_table, table_width, nh, 1.f, window, only_single,
                                 lse2, sums);
  return yalis_launch(only_single ? packed_sums_of_scores_kernel<true> : packed_sums_of_scores_kernel<false>,
                      dim3((unsigned)((max_kv_len + 255LL) / 256), g, n_requests), dim3(256), 0, stream, p, (const float*)scores, score_stride);
}

YALIS_SLOTS(yalis_packed_weight_sums)
YALIS_SLOTS(yalis_packed_sums_of_scores)
