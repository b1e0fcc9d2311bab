// Sums of attention weights per cached token for portions of prompts, on the 5th-generation tensor cores (head sizes 64 and 128).
//
// What packed_weight_sums.cu says, from keys that were unpacked for the prompt kernel (exact bfloat16 rows, see packed_rows.cu) and the
// logarithms that kernel left: A_j += sum over rows n and heads of 2^(scale q_n . k_j - lse2_n).  A work item is 128 keys of a KV head
// of a request; it walks the tiles of up to 128 query rows (token, head) that see any of them:
//
//   S^T = K Q^T    tcgen05.mma, K and Q tiles in 128B-swizzled shared memory by TMA, S^T in tensor memory: a lane is a key, a column
//                  a query row;
//   A  += 2^(.)    three groups of four warps take the tiles in turn, each group with a buffer of its own in tensor memory, one thread
//                  per key: its 128 scores, less the rows' logarithms (from shared memory, the same for every lane), raised and
//                  added up in float32.  A warp fetches the logarithms for itself and meets no other.
//
// The rows of an item are divided into parts of as many tiles (keys at a prompt's start are seen by all of its rows, those at its end
// by few), which the resident blocks (one to an SM) draw from a counter, early keys first.  A warp leaves its share of a
// part (its 32 keys, every third tile from the first, second or third on) in scratch memory, and the last share of the keys to be done (a
// counter, at zero before) adds them in their order to memory, so that no order of arrival shows.  One warp draws parts, works out what
// they are for the others and issues the copies, one the products.
// Bound by the exponentials, 16 a cycle and SM: 1,024 cycles a tile, of 1,690 that a tile takes (a prompt of 8,192 tokens, 32 heads of 64
// over 8: 414 us; 2,048 tokens: 43 us, of which the start of the pipeline is a fifth).  One group: 1,660 cycles of waits in a row for
// every tile of a block, and a block per item left half of the time to the one with the most rows.
// All waits are bounded (error word, tensor memory freed).
#include "packed.cuh"
#include "slots.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int kKeys = 128, kRows = 128;
constexpr int kGroups = 3;        // of four warps that add up; as many tiles are under way (four groups: too few registers to fetch ahead)
constexpr int kCopyWarp = 4 * kGroups, kProductWarp = kCopyWarp + 1, kThreads = (kProductWarp + 1) * 32;
constexpr int kTmemColumns = 512;  // a power of two that holds kGroups * kRows

struct SumsParams {
  const int32_t* positions;    // [N]
  const int32_t* q_start;      // [R + 1]
  const int32_t* block_table;  // [R, table_width] of the packed pages
  int table_width, n_requests, nh, per, window, skip_single;
  int width;                   // pages of 64 keys that a request has in the unpacked pool
  int rows_per_tile, tokens_per_tile, n_items;
  int parts, each;               // most parts of an item's rows, tiles of a part; index = item * parts + part
  float* partial;                // [items, parts, kGroups, 128]
  int32_t* counters;             // [1 + 4 items] the next part to draw; shares that are done of each 32 keys of an item; zero before
  float scale_log2;
  const float* lse2;           // [N, nh]
  float* sums;                 // [pages, g, page_size]
  int32_t* error;
  PackedPages pages;
};

// What a part is, as the copy warp hands it to the others.
struct Item {
  int req, kvh, key0;
  int tok0, begin, last, first;  // first row of the request, its place; the last place, and the first key that any row sees
  int t_lo, t_hi;                // rows (tokens) of the part that see a key of the item
  int item, part;                // the item's number, and which part of its rows this is (item -1: no more)
  int n_tiles, parts;            // tiles of the part; parts that have rows
  int each_shares, last_shares;  // groups with tiles in every part but the last, and in the last
};

__device__ __forceinline__ bool item_of(const SumsParams& p, int index, Item& it) {
  it.item = index / p.parts;
  it.part = index - it.item * p.parts;
  it.kvh = it.item % p.pages.g;
  const int rest = it.item / p.pages.g;
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
  if (it.t_lo >= it.t_hi) return false;
  const int tiles = (it.t_hi - it.t_lo + p.tokens_per_tile - 1) / p.tokens_per_tile, each = p.each;
  const int parts = (tiles + each - 1) / each, rest_tiles = tiles - (parts - 1) * each;
  if (it.part >= parts) return false;
  it.n_tiles = it.part + 1 < parts ? each : rest_tiles;
  it.parts = parts;
  it.each_shares = min(kGroups, each);
  it.last_shares = min(kGroups, rest_tiles);
  it.t_lo += it.part * each * p.tokens_per_tile;
  it.t_hi = min(it.t_hi, it.t_lo + each * p.tokens_per_tile);
  return true;
}

template <int HS>
__global__ void __launch_bounds__(kThreads, 1)
packed_sums_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const SumsParams p) {
  constexpr int H2 = HS / 64, TILE_BYTES = 128 * HS * 2;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* k_s = base;                       // [2][H2][128 keys][128 B]
  unsigned char* q_s = k_s + 2 * TILE_BYTES;       // [kGroups][H2][128 rows][128 B]
  // (arrays of their own: through the pointer above the compiler loads them as if they could lie anywhere, at twice the time)
  __shared__ __align__(16) float lse_s[4 * kGroups][kRows];            // the rows' logarithms, every warp's own
  __shared__ __align__(16) int token_s[kRows];                         // token of a row within its tile
  __shared__ Item drawn_s[2];                      // parts drawn
  uint64_t* k_full = reinterpret_cast<uint64_t*>(q_s + kGroups * TILE_BYTES);       // 2
  uint64_t* k_empty = k_full + 2;                  // 2
  uint64_t* q_full = k_full + 4;                   // kGroups
  uint64_t* q_empty = q_full + kGroups;            // kGroups
  uint64_t* s_full = q_empty + kGroups;            // kGroups
  uint64_t* s_empty = s_full + kGroups;            // kGroups
  uint64_t* drawn_full = s_empty + kGroups;        // 2
  uint64_t* drawn_empty = drawn_full + 2;          // 2
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drawn_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&k_full[b], 1); mbar_init(&k_empty[b], 1);
      mbar_init(&drawn_full[b], 1); mbar_init(&drawn_empty[b], 1 + 4 * kGroups);
    }
    for (int b = 0; b < kGroups; ++b) {
      mbar_init(&q_full[b], 1); mbar_init(&q_empty[b], 1);
      mbar_init(&s_full[b], 1); mbar_init(&s_empty[b], 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Rows of a tile that no copy writes (heads that do not divide 128) stay zero, so that their scores are numbers.
  for (int i = threadIdx.x; i < kGroups * TILE_BYTES / 16; i += kThreads) reinterpret_cast<uint4*>(q_s)[i] = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  if (threadIdx.x < kRows) token_s[threadIdx.x] = (int)threadIdx.x < p.rows_per_tile ? (int)threadIdx.x / p.per : 0x40000000;
  if (warp == kProductWarp) {
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

  if (warp == kCopyWarp) {
    // ---- copies ----
    if (lane == 0) {
      bool ok = true;
      Item it;
      for (int n = 0; ok; ++n) {
        int index;
        do {
          index = atomicAdd(p.counters, 1);
        } while (index < p.n_items * p.parts && !item_of(p, index, it));
        if (index >= p.n_items * p.parts) it.item = -1;
        if (!mbar_wait(&drawn_empty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag)) break;
        drawn_s[n & 1] = it;
        mbar_arrive(&drawn_full[n & 1]);
        if (it.item < 0) break;
        const int kb = k_armed & 1;
        if (!mbar_wait(&k_empty[kb], ((k_armed >> 1) & 1) ^ 1, abort_flag)) break;
        mbar_expect_tx(&k_full[kb], TILE_BYTES);
        for (int h = 0; h < H2; ++h)
          for (int b = 0; b < 2; ++b) {            // (a page past the pool, or of the next request, fills rows that nobody reads)
            const int page = it.req * p.width + (it.key0 >> 6) + b;
            tma_load_2d(k_s + kb * TILE_BYTES + h * (kKeys * 128) + b * (64 * 128), &map_k, h * 64, (page * p.pages.g + it.kvh) * 64, &k_full[kb]);
          }
        ++k_armed;
        for (int t = it.t_lo; t < it.t_hi; t += p.tokens_per_tile) {
          const int b = q_armed % kGroups;
          if (!mbar_wait(&q_empty[b], ((q_armed / kGroups) & 1) ^ 1, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&q_full[b], (uint32_t)p.rows_per_tile * HS * 2);
          for (int h = 0; h < H2; ++h)
            tma_load_3d(q_s + b * TILE_BYTES + h * (kRows * 128), &map_q, h * 64, it.kvh * p.per, it.tok0 + t, &q_full[b]);
          ++q_armed;
        }
      }
    }
    __syncwarp();
  } else if (warp == kProductWarp) {
    // ---- products: the whole warp runs the loop, the elected lane issues ----
    const uint32_t elected = elect_one(), idesc = idesc_f16(kKeys, kRows, false);
    const uint64_t k_desc0 = desc_kmajor(smem_u32(k_s)), q_desc0 = desc_kmajor(smem_u32(q_s));
    uint32_t T = 0, n = 0;
    bool ok = true;
    Item it;
    while (ok) {
      const int kb = n & 1;
      if (!mbar_wait(&drawn_full[kb], (n >> 1) & 1, abort_flag)) break;
      it = drawn_s[kb];
      __syncwarp();
      if (lane == 0) mbar_arrive(&drawn_empty[kb]);
      if (it.item < 0) break;
      if (!mbar_wait(&k_full[kb], (n >> 1) & 1, abort_flag)) break;
      const uint64_t k_desc = k_desc0 + (uint64_t)((kb * TILE_BYTES) >> 4);
      for (int i = 0; i < it.n_tiles; ++i, ++T) {
        const int b = T % kGroups;
        const uint32_t ph = (T / kGroups) & 1;
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
        if (i == it.n_tiles - 1) umma_commit(elected, &k_empty[kb]);       // the last reader of these keys
      }
      ++n;
    }
    __syncwarp();
  } else {
    // ---- sums, one thread per key; this warp takes every kGroups-th tile ----
    const int group = warp >> 2, part32 = warp & 3;
    const uint32_t s_addr = tmem + ((uint32_t)(part32 * 32) << 16) + group * kRows;
    const uint64_t scale2 = pack2(-p.scale_log2, -p.scale_log2);
    long long row_off[4];                                                          // logarithms of rows 4 lane ... 4 lane + 3
    int token_of[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = 4 * lane + j;
      token_of[j] = row < p.rows_per_tile ? row / p.per : 0x40000000;
      row_off[j] = row < p.rows_per_tile ? (long long)(row / p.per) * p.nh + row % p.per : 0;
    }
    uint32_t T = 0, mine = 0;                                                      // tiles of the block, of this group
    Item it;
    for (int n = 0;; ++n) {
      if (!warp_wait(&drawn_full[n & 1], (n >> 1) & 1, abort_flag, lane)) break;
      it = drawn_s[n & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&drawn_empty[n & 1]);
      if (it.item < 0) break;
      const int key_lo = it.key0 + part32 * 32, key = key_lo + lane;
      float lse[4];
      auto fetch = [&](int t) {
        const float* from = p.lse2 + (size_t)(it.tok0 + t) * p.nh + it.kvh * p.per;
#pragma unroll
        for (int j = 0; j < 4; ++j) lse[j] = t + token_of[j] < it.t_hi ? from[row_off[j]] : INFINITY;
      };
      const int first_tile = (int)((group + kGroups - T % kGroups) % kGroups);     // tile i of the part is the block's tile T + i
      if (first_tile < it.n_tiles) fetch(it.t_lo + first_tile * p.tokens_per_tile);
      uint64_t sum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
      bool ok = true;
      for (int i = first_tile; i < it.n_tiles; i += kGroups, ++mine) {
        const int t = it.t_lo + i * p.tokens_per_tile, n_tok = min(p.tokens_per_tile, it.t_hi - t);
        const int place = it.begin + t, last_place = it.begin + (t + n_tok - 1);
        *reinterpret_cast<float4*>(&lse_s[warp][4 * lane]) = make_float4(lse[0], lse[1], lse[2], lse[3]);
        __syncwarp();
        if (i + kGroups < it.n_tiles) fetch(t + kGroups * p.tokens_per_tile);
        if (!warp_wait(&s_full[group], mine & 1, abort_flag, lane)) { ok = false; break; }
        if (last_place >= key_lo) {                // (else no row of the tile sees a key of this warp)
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const bool masked = n_tok < p.tokens_per_tile || place < key_lo + 31 || (p.window > 0 && last_place - p.window >= key_lo);
          // Row c sees this lane's key if lowest <= token < beyond.
          const int lowest = key - it.begin - t, beyond = p.window > 0 ? (int)min((long long)n_tok, (long long)lowest + p.window) : n_tok;
          auto add = [&](const float (&s)[32], int c0) {
            const float4* lse4 = reinterpret_cast<const float4*>(&lse_s[warp][c0]);
            if (masked) {
              const int4* token4 = reinterpret_cast<const int4*>(&token_s[c0]);
#pragma unroll
              for (int c = 0; c < 32; c += 4) {
                const float4 off = lse4[c / 4];
                const int4 at = token4[c / 4];
                auto one = [&](float v, float o, int token) {
                  const float e = ex2(fmaf(v, p.scale_log2, -o));
                  return token >= lowest && token < beyond ? e : 0.f;
                };
                sum2[0] = add2(sum2[0], pack2(one(s[c], off.x, at.x), one(s[c + 1], off.y, at.y)));
                sum2[1] = add2(sum2[1], pack2(one(s[c + 2], off.z, at.z), one(s[c + 3], off.w, at.w)));
              }
            } else {
#pragma unroll
              for (int c = 0; c < 32; c += 4) {
                const float4 off = lse4[c / 4];
                float x0, x1, x2, x3;              // the logarithm less the score
                unpack2(fma2(pack2(s[c], s[c + 1]), scale2, pack2(off.x, off.y)), x0, x1);
                unpack2(fma2(pack2(s[c + 2], s[c + 3]), scale2, pack2(off.z, off.w)), x2, x3);
                sum2[0] = add2(sum2[0], pack2(ex2(-x0), ex2(-x1)));
                sum2[1] = add2(sum2[1], pack2(ex2(-x2), ex2(-x3)));
              }
            }
          };
          // 32 scores are on their way while the 32 before are added
          float sa[32], sb[32];
          __syncwarp();
          tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&sa[0]));
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&sb[0]));
          add(sa, 0);
          __syncwarp();
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          tmem_ld32(s_addr + 64, *reinterpret_cast<uint32_t(*)[32]>(&sa[0]));
          add(sb, 32);
          __syncwarp();
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          tmem_ld32(s_addr + 96, *reinterpret_cast<uint32_t(*)[32]>(&sb[0]));
          add(sa, 64);
          __syncwarp();
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[group]);       // the products may write the next tile's scores
          add(sb, 96);
        } else if (lane == 0) {
          mbar_arrive(&s_empty[group]);
        }
        __syncwarp();                              // the logarithms have been read
      }
      if (!ok) break;
      T += (uint32_t)it.n_tiles;
      if (first_tile >= it.n_tiles) continue;
      float a, b, c, d;
      unpack2(sum2[0], a, b);
      unpack2(sum2[1], c, d);
      float total = (a + b) + (c + d);
      const int shares = (it.parts - 1) * it.each_shares + it.last_shares;
      if (shares > 1) {
        float* partial = p.partial + (size_t)it.item * p.parts * kGroups * kKeys + part32 * 32 + lane;
        partial[(size_t)(it.part * kGroups + first_tile) * kKeys] = total;
        __threadfence();
        __syncwarp();
        int last = 0;
        if (lane == 0) last = atomicAdd(p.counters + 1 + it.item * 4 + part32, 1) == shares - 1;
        if (!__shfl_sync(0xffffffffu, last, 0)) continue;
        __threadfence();
        total = 0.f;
        for (int i = 0; i < it.parts; ++i)
          for (int k = 0; k < (i + 1 < it.parts ? it.each_shares : it.last_shares); ++k)
            total += __ldcg(partial + (size_t)(i * kGroups + k) * kKeys);
      }
      if (key > it.last || key < it.first) continue;
      int row;
      const int page = page_of(p.pages, p.block_table + (size_t)it.req * p.table_width, p.table_width, key, row);
      if (page >= 0) atomicAdd(p.sums + row_index(p.pages, page, it.kvh, row), total);
    }
    __syncwarp();
  }

  // ---- exit: drain on abort, free tensor memory ----
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == kCopyWarp * 32) {
      if (p.error) atomicOr(p.error, YALIS_FLAG_WAIT_ATTENTION);
      for (int j = max(0, k_armed - 2); j < k_armed; ++j)
        for (uint32_t i = 0; i < kSpinLimit; ++i)
          if (mbar_try_wait(&k_full[j & 1], (j >> 1) & 1)) break;
      for (int j = max(0, q_armed - kGroups); j < q_armed; ++j)
        for (uint32_t i = 0; i < kSpinLimit; ++i)
          if (mbar_try_wait(&q_full[j % kGroups], (j / kGroups) & 1)) break;
    }
    __syncthreads();
  }
  if (warp == kProductWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
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
  const size_t smem = 1024 + (2 + kGroups) * 128 * HS * 2 + (8 + 4 * kGroups) * 8 + 8;
  static bool configured[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return YALIS_ERR_LAUNCH;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(packed_sums_tcgen05_kernel<HS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return YALIS_ERR_LAUNCH;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int units = p.n_items * p.parts, grid = units < yalis_sm_count() ? units : yalis_sm_count();
  return yalis_launch(packed_sums_tcgen05_kernel<HS>, dim3(grid), dim3(kThreads), smem, stream, mq, mk, p);
}

}  // namespace

// k_unpacked: [n_requests * width, g, 64, dim] bfloat16 (yalis_packed_unpack).  q rows on 16-byte boundaries.  With items =
// ceil(max_kv_len / 128) * n_requests * g, an item's rows go in up to `parts` parts of `each` tiles (all of them): partial [items, parts, 3, 128] floats, counters [1 + 4 items] at zero.
YALIS_API int yalis_packed_sums_tcgen05(const void* q, long long q_stride, const void* k_unpacked, int width, int num_pages, int page_size, int g,
                                        int dim, const int32_t* positions, const int32_t* q_start, const int32_t* block_table, int table_width,
                                        int n_requests, int n_tokens, int max_kv_len, int nh, float scale, int window, int skip_single,
                                        float* lse2, float* sums, int each, int parts, float* partial, int32_t* counters, int32_t* error, cudaStream_t stream) {
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
  if (parts < 1 || each < 1 || items * parts > 0x7fffffffll || rows + (long long)g * 64 > 0x7fffffffll) return YALIS_ERR_SHAPE;
  p.n_items = (int)items; p.parts = parts; p.each = each; p.partial = partial; p.counters = counters;
  p.scale_log2 = scale * 1.4426950408889634f; p.lse2 = lse2; p.sums = sums; p.error = error;
  p.pages = packed_pages(nullptr, nullptr, nullptr, num_pages, page_size, g, dim);
  CUtensorMap mq, mk;
  const cuuint64_t q_sizes[3] = {(cuuint64_t)dim, (cuuint64_t)nh, (cuuint64_t)n_tokens}, q_strides[2] = {(cuuint64_t)dim * 2, (cuuint64_t)q_stride * 2};
  const cuuint32_t q_box[3] = {64u, (cuuint32_t)per, (cuuint32_t)p.tokens_per_tile};
  const cuuint64_t k_sizes[2] = {(cuuint64_t)dim, (cuuint64_t)rows}, k_strides[1] = {(cuuint64_t)dim * 2};
  const cuuint32_t k_box[2] = {64u, 64u};
  if (!encode(&mq, 3, q, q_sizes, q_strides, q_box) || !encode(&mk, 2, k_unpacked, k_sizes, k_strides, k_box)) return YALIS_ERR_LAUNCH;
  return dim == 64 ? launch_sums<64>(mq, mk, p, stream) : launch_sums<128>(mq, mk, p, stream);
}

YALIS_SLOTS(yalis_packed_sums_tcgen05)
