// Sums of attention weights per cached token for portions of prompts, on the 5th-generation tensor cores (head sizes 64 and 128).
//
// What packed_weight_sums.cu says, from keys that were unpacked for the prompt kernel (exact bfloat16 rows, see packed_rows.cu) and the
// logarithms that kernel left: A_j += sum over rows n and heads of 2^(scale q_n . k_j - lse2_n).  A work item is 128 keys of a KV head
// of a request; it walks the tiles of up to 128 query rows (token, head) that see any of them:
//
//   S^T = K Q^T    tcgen05.mma, K and Q tiles in 128B-swizzled shared memory by TMA, S^T in tensor memory, double buffered: a lane
//                  is a key, a column a query row;
//   A  += 2^(.)    four warps, one thread per key: its 128 scores from tensor memory, less the rows' logarithms (from shared memory,
//                  the same for every lane), raised and added up in float32.
//
// A key's sum never leaves its thread until the item's end, so there is one addition to memory per token and nothing whose order could
// change.  One warp issues the copies, one the products; items go round the resident blocks (two to an SM), those of early keys, which
// most rows see, first.  Bound by the softmax warps' instructions (2.5 a score) as much as by the exponentials.
// All waits are bounded (error word, tensor memory freed).
#include "packed.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int kKeys = 128, kRows = 128;
constexpr int kThreads = 192;     // warps 0-3 sums, warp 4 copies, warp 5 products + tensor memory
constexpr int kTmemColumns = 256; // two S^T of 128 columns

struct SumsParams {
  const int32_t* positions;    // [N]
  const int32_t* q_start;      // [R + 1]
  const int32_t* block_table;  // [R, table_width] of the packed pages
  int table_width, n_requests, nh, per, window, skip_single;
  int width;                   // pages of 64 keys that a request has in the unpacked pool
  int rows_per_tile, tokens_per_tile, n_items;
  float scale_log2;
  const float* lse2;           // [N, nh]
  float* sums;                 // [pages, g, page_size]
  int32_t* error;
  PackedPages pages;
};

// What an item is; every role works it out for itself.
struct Item {
  int req, kvh, key0;
  int tok0, begin, last, first;  // first row of the request, its place; the last place, and the first key that any row sees
  int t_lo, t_hi;                // rows (tokens) that see a key of the item
};

__device__ __forceinline__ bool item_of(const SumsParams& p, int index, Item& it) {
  it.kvh = index % p.pages.g;
  const int rest = index / p.pages.g;
  it.req = rest % p.n_requests;
  it.key0 = rest / p.n_requests * kKeys;
  it.tok0 = p.q_start[it.req];
  const int n = p.q_start[it.req + 1] - it.tok0;
  if (n <= 0 || (p.skip_single && n == 1)) return false;
  it.begin = p.positions[it.tok0];
  it.last = p.positions[it.tok0 + n - 1];
  it.first = p.window > 0 ? max(0, it.begin - p.window + 1) : 0;
  if (it.key0 > it.last || it.key0 + kKeys <= it.first) return false;
  it.t_lo = min(max(it.key0 - it.begin, 0), n);
  it.t_hi = p.window > 0 ? (int)min((long long)n, max(0ll, (long long)it.key0 + kKeys - 1 + p.window - it.begin)) : n;
  return it.t_lo < it.t_hi;
}

template <int HS>
__global__ void __launch_bounds__(kThreads, 2)
packed_sums_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const SumsParams p) {
  constexpr int H2 = HS / 64, TILE_BYTES = 128 * HS * 2;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* k_s = base;                       // [H2][128 keys][128 B]
  unsigned char* q_s = k_s + TILE_BYTES;           // [2][H2][128 rows][128 B]
  float* less_s = reinterpret_cast<float*>(q_s + 2 * TILE_BYTES);      // [2][128] minus the rows' logarithms
  int* place_s = reinterpret_cast<int*>(less_s + 2 * kRows);           // [2][128] the rows' places, -1: no row
  uint64_t* k_full = reinterpret_cast<uint64_t*>(place_s + 2 * kRows);
  uint64_t* k_empty = k_full + 1;
  uint64_t* q_full = k_full + 2;                   // 2
  uint64_t* q_empty = k_full + 4;                  // 2
  uint64_t* s_full = k_full + 6;                   // 2
  uint64_t* s_empty = k_full + 8;                  // 2
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(k_full + 10);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    mbar_init(k_empty, 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&q_full[b], 1); mbar_init(&q_empty[b], 1);
      mbar_init(&s_full[b], 1); mbar_init(&s_empty[b], 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Rows of a tile that no copy writes (heads that do not divide 128) stay zero, so that their scores are numbers.
  for (int i = threadIdx.x; i < 2 * TILE_BYTES / 16; i += kThreads) reinterpret_cast<uint4*>(q_s)[i] = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemColumns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tmem = *tmem_slot;
  int k_armed = 0, q_armed = 0;                    // copies asked for (for the drain)

  if (warp == 4) {
    // ---- copies ----
    if (lane == 0) {
      bool ok = true;
      Item it;
      for (int index = blockIdx.x; ok && index < p.n_items; index += gridDim.x) {
        if (!item_of(p, index, it)) continue;
        if (!mbar_wait(k_empty, (k_armed & 1) ^ 1, abort_flag)) break;
        mbar_expect_tx(k_full, TILE_BYTES);
        for (int h = 0; h < H2; ++h)
          for (int b = 0; b < 2; ++b) {            // (a page past the pool, or of the next request, fills rows that nobody reads)
            const int page = it.req * p.width + (it.key0 >> 6) + b;
            tma_load_2d(k_s + h * (kKeys * 128) + b * (64 * 128), &map_k, h * 64, (page * p.pages.g + it.kvh) * 64, k_full);
          }
        ++k_armed;
        for (int t = it.t_lo; t < it.t_hi; t += p.tokens_per_tile) {
          const int b = q_armed & 1;
          if (!mbar_wait(&q_empty[b], ((q_armed >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&q_full[b], (uint32_t)p.rows_per_tile * HS * 2);
          for (int h = 0; h < H2; ++h)
            tma_load_3d(q_s + b * TILE_BYTES + h * (kRows * 128), &map_q, h * 64, it.kvh * p.per, it.tok0 + t, &q_full[b]);
          ++q_armed;
        }
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    // ---- products: the whole warp runs the loop, the elected lane issues ----
    const uint32_t elected = elect_one(), idesc = idesc_f16(kKeys, kRows, false);
    const uint64_t k_desc = desc_kmajor(smem_u32(k_s)), q_desc0 = desc_kmajor(smem_u32(q_s));
    uint32_t T = 0, n = 0;
    bool ok = true;
    Item it;
    for (int index = blockIdx.x; ok && index < p.n_items; index += gridDim.x) {
      if (!item_of(p, index, it)) continue;
      if (!mbar_wait(k_full, n & 1, abort_flag)) break;
      for (int t = it.t_lo; t < it.t_hi; t += p.tokens_per_tile, ++T) {
        const int b = T & 1;
        const uint32_t ph = (T >> 1) & 1;
        if (!mbar_wait(&q_full[b], ph, abort_flag) || !mbar_wait(&s_empty[b], ph ^ 1, abort_flag)) { ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t q_desc = q_desc0 + (uint64_t)((b * TILE_BYTES) >> 4);
#pragma unroll
        for (int ks = 0; ks < HS / 16; ++ks) {
          const uint32_t off = (ks >> 2) * (128 * 128) + (ks & 3) * 32;
          umma_ss(elected, tmem + b * kRows, k_desc + (off >> 4), q_desc + (off >> 4), idesc, ks > 0);
        }
        umma_commit(elected, &s_full[b]);
        umma_commit(elected, &q_empty[b]);
        if (t + p.tokens_per_tile >= it.t_hi) umma_commit(elected, k_empty);       // the last reader of these keys
      }
      ++n;
    }
    __syncwarp();
  } else {
    // ---- sums, one thread per key ----
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
    const int t_in = threadIdx.x / p.per, h_in = threadIdx.x - t_in * p.per;       // the row that this thread describes
    uint32_t T = 0;
    bool ok = true;
    Item it;
    // (after a wait that ran out the warps still go through the loops, so that they keep meeting, but wait and add no more)
    for (int index = blockIdx.x; index < p.n_items; index += gridDim.x) {
      if (!item_of(p, index, it)) continue;
      const int key = it.key0 + threadIdx.x, key_lo = it.key0 + warp * 32;
      int row, page = -1;
      if (key <= it.last && key >= it.first) page = page_of(p.pages, p.block_table + (size_t)it.req * p.table_width, p.table_width, key, row);
      float less = -INFINITY;
      int place = -1;
      auto describe = [&](int t) {
        const bool real = t + t_in < it.t_hi && (int)threadIdx.x < p.rows_per_tile;
        less = real ? -p.lse2[(size_t)(it.tok0 + t + t_in) * p.nh + it.kvh * p.per + h_in] : -INFINITY;
        place = real ? p.positions[it.tok0 + t + t_in] : -1;
      };
      describe(it.t_lo);
      uint64_t sum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
      for (int t = it.t_lo; t < it.t_hi; t += p.tokens_per_tile, ++T) {
        const int b = T & 1;
        less_s[b * kRows + threadIdx.x] = less;
        place_s[b * kRows + threadIdx.x] = place;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (t + p.tokens_per_tile < it.t_hi) describe(t + p.tokens_per_tile);
        const int n_tok = min(p.tokens_per_tile, it.t_hi - t);
        const bool masked = n_tok < p.tokens_per_tile || it.begin + t < key_lo + 31 ||
                            (p.window > 0 && it.begin + t + n_tok - 1 - p.window >= key_lo);
        if (ok) ok = warp_wait(&s_full[b], (T >> 1) & 1, abort_flag, lane);
        if (!ok) continue;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
        for (int c0 = 0; c0 < kRows; c0 += 64) {
          float s[64];
          __syncwarp();
          tmem_ld32(lane_base + b * kRows + c0, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
          tmem_ld32(lane_base + b * kRows + c0 + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          const float4* less4 = reinterpret_cast<const float4*>(less_s + b * kRows + c0);
          if (masked) {
            const int4* place4 = reinterpret_cast<const int4*>(place_s + b * kRows + c0);
#pragma unroll
            for (int c = 0; c < 64; c += 4) {
              const float4 off = less4[c / 4];
              const int4 at = place4[c / 4];
              auto one = [&](float v, float o, int w) {
                const float e = ex2(fmaf(v, p.scale_log2, o));
                return key <= w && !(p.window > 0 && key <= w - p.window) ? e : 0.f;
              };
              sum2[0] = add2(sum2[0], pack2(one(s[c], off.x, at.x), one(s[c + 1], off.y, at.y)));
              sum2[1] = add2(sum2[1], pack2(one(s[c + 2], off.z, at.z), one(s[c + 3], off.w, at.w)));
            }
          } else {
#pragma unroll
            for (int c = 0; c < 64; c += 4) {
              const float4 off = less4[c / 4];
              float x0, x1, x2, x3;
              unpack2(fma2(pack2(s[c], s[c + 1]), scale2, pack2(off.x, off.y)), x0, x1);
              unpack2(fma2(pack2(s[c + 2], s[c + 3]), scale2, pack2(off.z, off.w)), x2, x3);
              sum2[0] = add2(sum2[0], pack2(ex2(x0), ex2(x1)));
              sum2[1] = add2(sum2[1], pack2(ex2(x2), ex2(x3)));
            }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[b]);
      }
      if (ok && page >= 0) {
        float a, b, c, d;
        unpack2(sum2[0], a, b);
        unpack2(sum2[1], c, d);
        atomicAdd(p.sums + row_index(p.pages, page, it.kvh, row), (a + b) + (c + d));
      }
    }
  }

  // ---- exit: drain on abort, free tensor memory ----
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 4 * 32) {
      if (p.error) atomicOr(p.error, YALIS_FLAG_WAIT_ATTENTION);
      if (k_armed > 0)
        for (uint32_t i = 0; i < kSpinLimit; ++i)
          if (mbar_try_wait(k_full, (k_armed - 1) & 1)) break;
      for (int j = max(0, q_armed - 2); j < q_armed; ++j)
        for (uint32_t i = 0; i < kSpinLimit; ++i)
          if (mbar_try_wait(&q_full[j & 1], (j >> 1) & 1)) break;
    }
    __syncthreads();
  }
  if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
}

bool encode(CUtensorMap* map, int dims, const void* at, const cuuint64_t* sizes, const cuuint64_t* strides, const cuuint32_t* box) {
  EncodeTiledFn fn = encode_fn();
  const cuuint32_t ones[3] = {1, 1, 1};
  return fn != nullptr && fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)dims, const_cast<void*>(at), sizes, strides, box, ones,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HS>
int launch_sums(const CUtensorMap& mq, const CUtensorMap& mk, const SumsParams& p, cudaStream_t stream) {
  const size_t smem = 1024 + 3 * 128 * HS * 2 + 4 * kRows * 4 + 10 * 8 + 8;
  static bool configured[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return YALIS_ERR_LAUNCH;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(packed_sums_tcgen05_kernel<HS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return YALIS_ERR_LAUNCH;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int grid = p.n_items < 2 * yalis_sm_count() ? p.n_items : 2 * yalis_sm_count();
  return yalis_launch(packed_sums_tcgen05_kernel<HS>, dim3(grid), dim3(kThreads), smem, stream, mq, mk, p);
}

}  // namespace

// k_unpacked: [n_requests * width, g, 64, dim] bfloat16 (yalis_packed_unpack).  q rows on 16-byte boundaries.
YALIS_API int yalis_packed_sums_tcgen05(const void* q, long long q_stride, const void* k_unpacked, int width, int num_pages, int page_size, int g,
                                        int dim, const int32_t* positions, const int32_t* q_start, const int32_t* block_table, int table_width,
                                        int n_requests, int n_tokens, int max_kv_len, int nh, float scale, int window, int skip_single,
                                        float* lse2, float* sums, int32_t* error, cudaStream_t stream) {
  if ((dim != 64 && dim != 128) || g < 1 || nh % g || nh / g > 128 || page_size < 1) return YALIS_ERR_SHAPE;
  if (n_requests <= 0 || n_tokens <= 0 || max_kv_len <= 0) return YALIS_OK;
  if ((((uintptr_t)q | (uintptr_t)k_unpacked) & 15) || (q_stride % 8)) return YALIS_ERR_ALIGN;
  const int per = nh / g;
  SumsParams p = {};
  p.positions = positions; p.q_start = q_start; p.block_table = block_table; p.table_width = table_width; p.n_requests = n_requests;
  p.nh = nh; p.per = per; p.window = window; p.skip_single = skip_single; p.width = width;
  p.tokens_per_tile = kRows / per; p.rows_per_tile = p.tokens_per_tile * per;
  const long long items = (long long)((max_kv_len + kKeys - 1) / kKeys) * n_requests * g;
  const long long rows = (long long)n_requests * width * g * 64;
  if (items > 0x7fffffffll || rows + (long long)g * 64 > 0x7fffffffll) return YALIS_ERR_SHAPE;
  p.n_items = (int)items;
  p.scale_log2 = scale * 1.4426950408889634f; p.lse2 = lse2; p.sums = sums; p.error = error;
  p.pages = {nullptr, nullptr, nullptr, num_pages, page_size, g, dim};
  CUtensorMap mq, mk;
  const cuuint64_t q_sizes[3] = {(cuuint64_t)dim, (cuuint64_t)nh, (cuuint64_t)n_tokens}, q_strides[2] = {(cuuint64_t)dim * 2, (cuuint64_t)q_stride * 2};
  const cuuint32_t q_box[3] = {64u, (cuuint32_t)per, (cuuint32_t)p.tokens_per_tile};
  const cuuint64_t k_sizes[2] = {(cuuint64_t)dim, (cuuint64_t)rows}, k_strides[1] = {(cuuint64_t)dim * 2};
  const cuuint32_t k_box[2] = {64u, 64u};
  if (!encode(&mq, 3, q, q_sizes, q_strides, q_box) || !encode(&mk, 2, k_unpacked, k_sizes, k_strides, k_box)) return YALIS_ERR_LAUNCH;
  return dim == 64 ? launch_sums<64>(mq, mk, p, stream) : launch_sums<128>(mq, mk, p, stream);
}
