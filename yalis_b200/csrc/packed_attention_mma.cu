// Attention over pages held in 4 bits (packed.cuh) on the tensor cores, for single tokens and short portions in bfloat16 and for
// every step in float32 (head sizes 64 and 128).  What is computed is what packed_attention.cu says.
//
// A pair is a KV head of a request with up to 8 NT of its query rows (row = token * heads per KV head + head), which are the columns
// here: both products are taken transposed, so that the codes are the operand of 16 rows and a lane turns the codes it has loaded
// into pairs of numbers in registers, with nothing in between:
//
//   S^T [keys, columns] = C_K [16 keys x 16 elements] q^T       O^T [elements, columns] += C_V^T [16 elements x 16 keys] W^T
//
// The order of a product's inner index is free as long as both operands agree, so a lane takes neighbouring codes.
//
// bfloat16 queries: both products are taken in float16, where a code needs nothing but a mask.  Four bits c at the bottom of a 16-bit half
// are the float16 number c 2^-24, the next four c 2^-20 (numbers below 2^-14 are linear in their bits), so two of a half word's four codes
// need no shift.  Zeros are multiplied out apart: for keys zero sum(q) is taken from the product, for values the weights' product with the
// zeros (a tile of its own) from the output, in place of 64 subtractions a chunk each.  Queries go in by a power of two that puts a row's
// largest near the top of float16, which loses no bit of anything above 2^-28 of it; weights keep eleven bits: every column's exponentials
// are taken relative to its largest weight times value's step so far instead of its largest weight, so that a key that a column does not
// see, or gives no weight, has no say in how its others are rounded.
// float32 queries: codes become bfloat16 pairs, with a word of eight codes (w >> s) & 0x00780078 | 0x41804180 is 16 + c_i, 16 + c_(i + 4),
// less 16 + zero; queries and weights go in as three bfloat16 parts (sums of large numbers that cancel would show here).
// Elements of a V row pair up by key: the 16-bit halves of two keys' words are put side by side first.  The scores' accumulators, times
// step, are the softmax's scores; weights are turned from accumulator layout to operand layout by movmatrix.
//
// A warp takes 32 keys at a time (a chunk) through a ring of its own in shared memory, filled by 16-byte asynchronous copies, and
// keeps a softmax and an output of its own; the four warps of a block come together at the end of a pair.  Chunks are
// dealt to a fixed grid by the step's lengths (choose_deal), so that a recorded launch serves other lengths too; a pair cut between
// blocks is added up, in the blocks' order, by whichever of them comes last (a counter per pair, left at zero).  Nothing waits for
// another block.
// Bound by instructions, about 490 a chunk and warp (620 and 9 % more time with shifts and subtractions for every pair): 8 requests of
// 18,000 to 32,000 keys, 24 heads of 128 over 8: 58 us, 212 MB at 3.7 TB/s; 64 requests of 540 to 1,040, 32 heads: 23 us (the general
// form: 4,640 and 280).
#include <cuda_fp16.h>

#include <type_traits>

#include "packed.cuh"
#include "slots.cuh"

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kChunk = 32;     // keys of a chunk
constexpr int kStages = 2;
constexpr float kNone = -1e30f;  // the maximum of no scores
constexpr float kUnset = -3e38f; // limit of a column that has seen no score yet: any will do
constexpr float kLazy = 8.f;   // how far (log2) scores may rise above the maximum in use before the output is rescaled
constexpr float kTarget = 6.f; // where (log2) the largest weight times its value's step lies in float16 after that: below 2^15 with kLazy more
constexpr float kSmall = -80.f;  // steps of less (log2) count as this, which keeps the weights themselves within float32; so do those that are none

struct MmaParams {
  const void* q;               // [N, q_stride]
  long long q_stride;
  void* out;                   // [N, out_stride]
  long long out_stride;
  const int32_t* positions;    // [N]
  const int32_t* q_start;      // [R + 1]
  const int32_t* block_table;  // [R, table_width]
  int table_width, n_requests, nh, per, window;
  int reach;                   // places that the table has
  int together;                // 2: a chunk never lies in two pages; 1: the rows that one copy instruction of a warp covers do not
  int q_vector;                // 1: rows of q start on 16-byte boundaries
  int only_single;             // 1: requests that bring more than one token are left to another kernel
  int slots;                   // blocks resident at once; the launch has as many, or one for every pair
  float scale_log2;
  float* lse2;                 // [N, nh] the logarithm to base two of a row's sum of exponentials, or null
  float* scores;               // [N, nh, score_stride] every score in powers of two, by place (those that some row of the pair sees), or
                               // null; with only_single [R, nh, score_stride], a request's row
  long long score_stride;
  float* part;                 // [blocks, 2, MT * 32 * 4 + 16 NT * 2]
  int32_t* tickets;            // one per pair, zero before and after
  int32_t* error;
  PackedPages pages;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pair_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pair_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b) {
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 16 + codes i and i + 4 of the eight in w as bfloat16.
// One three-input operation: a register has to hold 16, 16 (an instruction takes one constant; with two written out the compiler
// made two instructions of it, which was a quarter of all that the kernel issued).
template <int I>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t sixteens) {
  const uint32_t at = I == 0 ? w << 3 : w >> (I == 0 ? 0 : 4 * I - 3);
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00780078, %2, 0xEA;" : "=r"(r) : "r"(at), "r"(sixteens));       // (at & mask) | sixteens
  return r;
}
// Parts of a float32 pair in bfloat16: PARTS 1 rounds it; 3 hold every bit.
template <int PARTS>
__device__ __forceinline__ void parts_of(float x, float y, uint32_t (&out)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    out[i] = pair_bf16(x, y);
    if (i + 1 < PARTS) {
      x -= __uint_as_float(out[i] << 16);
      y -= __uint_as_float(out[i] & 0xFFFF0000u);
    }
  }
}

// Which key of 16 stands in row i of a product's tile: rows 2t hold keys t, rows 2t + 1 keys 4 + (t ^ X), so that the lanes of a
// quarter (K) or half (V) of a warp read different banks.
template <int DIM>
__device__ __forceinline__ int key_of_row(int i) {
  constexpr int X = DIM == 128 ? 1 : 2;
  return (i & 8) + ((i & 1) ? 4 + (((i & 7) >> 1) ^ X) : (i & 7) >> 1);
}
// Byte of a chunk's row r (DIM / 2 bytes) in shared memory, in pieces of 16; rows of 64 bytes swap their halves every other pair.
template <int DIM>
__device__ __forceinline__ int piece_at(int r, int piece) {
  return r * (DIM / 2) + ((DIM == 128 ? piece ^ (r & 2) : piece) << 4);
}

template <int DIM>
struct Stage {
  unsigned char k[kChunk * DIM / 2];
  unsigned char v[kChunk * DIM / 2];
  uint32_t words[kChunk];
};

// What a key's word says, as the products with bfloat16 pairs use it: the key's step times scale, 16 + its zero, the value's step, 16 +
// its zero.
// A key that is not there has a value's step of 0 (a row that is there has at least 2^-126; times scale it may be 0).
__device__ __forceinline__ float4 terms_of(uint32_t word, float scale_log2) {
  return make_float4(step_of(word & 0xFFFFu) * scale_log2, __uint_as_float(0x41800000u | (word & 15u) << 19), step_of(word >> 16),
                     __uint_as_float(0x41800000u | (word >> 16 & 15u) << 19));
}

// How a step's chunks are dealt out, by what the slowest block then has to do, counted in chunks:
//   pieces k > 0: every pair to k blocks in equal pieces, one piece a block (one, where there are more pairs than blocks resident at
//   once: the rest follow as blocks end);
//   0: all chunks of all pairs, laid end to end, in equal shares; a block's share begins and ends inside pairs that others share.
// A piece is at least kLeast chunks; to come together with other blocks takes about kJoin chunks' time (64 requests of 540 to 1,040
// tokens, 8 KV heads of 128: 25 us whole, 36 in equal shares; 8 of 18,000 to 32,000: 66 in nine pieces, 69 in equal shares).
// More pairs than blocks go out whole, whatever their lengths, which is right where they are alike and short (whole / equal shares, us, heads
// of 128 over 8: 80 requests of 450 to 900 tokens 37 / 43, 128 of them 45 / 53, 200 of 100 to 300 43 / 53), not where they are long
// (128 of 2,000 to 8,000: 192 / 174) and least where one is (96 requests, one of 30,000, the others of 200 to 1,000: 269 / 60, in float32
// 327 / 83): one block walks each of its pairs.
struct Deal {
  int pieces, blocks;
};
constexpr int kLeast = 2 * kWarps, kJoin = 32;

__device__ __forceinline__ Deal choose_deal(int slots, int pairs, int most, long long total) {
  if (pairs > slots) return {1, pairs};
  const int even_blocks = (int)min((long long)slots, (total + kLeast - 1) / kLeast);
  const int k = max(1, min(slots / pairs, (most + kLeast - 1) / kLeast));
  const long long even = total / even_blocks + 2 * kJoin;
  if ((most + k - 1) / k + (k > 1 ? kJoin : 0) <= even) return {k, pairs * k};
  return {0, even_blocks};
}


// SCORES: every score is left in memory as well (a branch on the pointer in the one kernel cost 3 % of the steps that want none).
template <typename T, int DIM, int NT, int PARTS, bool SCORES>
__global__ void __launch_bounds__(kThreads, NT == 1 && PARTS == 1 ? 4 : 2) packed_attention_mma_kernel(const MmaParams p) {
  constexpr int W = DIM / 32;                  // words of a K row that a lane takes
  constexpr int U = DIM / 64;                  // words of a V row that a lane takes
  constexpr int MT = DIM / 16;                 // tiles of 16 elements of the output
  constexpr int COLS = 8 * NT;
  constexpr int PIECES = DIM / 32;             // 16-byte pieces of a row
  constexpr int COPIES = PIECES;               // of K (and as many of V) that a lane asks for per chunk
  constexpr int PART_FLOATS = NT * MT * 128 + 2 * COLS;
  constexpr bool HALF = PARTS == 1;            // products in float16
  extern __shared__ __align__(128) unsigned char smem[];
  Stage<DIM>* ring = reinterpret_cast<Stage<DIM>*>(smem) + (threadIdx.x >> 5) * kStages;
  float4* terms = reinterpret_cast<float4*>(smem + sizeof(Stage<DIM>) * kStages * kWarps) + (threadIdx.x >> 5) * kChunk;
  float* height = reinterpret_cast<float*>(smem + sizeof(Stage<DIM>) * kStages * kWarps + kWarps * kChunk * 16) + (threadIdx.x >> 5) * kChunk;
  float4* merge_o = reinterpret_cast<float4*>(smem + sizeof(Stage<DIM>) * kStages * kWarps + kWarps * kChunk * 20);   // [kWarps][NT * MT][32]
  float* merge_ml = reinterpret_cast<float*>(merge_o + kWarps * NT * MT * 32);                     // [kWarps][COLS][2]
  int* s_last = reinterpret_cast<int*>(merge_ml + kWarps * COLS * 2);
  int* s_deal = s_last + 1;                                                                        // pieces, blocks
  long long* cum = reinterpret_cast<long long*>(s_last + 4);                                       // [R + 1] chunks before request r
  int* cum_pairs = reinterpret_cast<int*>(cum + p.n_requests + 1);                                 // [R + 1] pairs before it

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t sixteens;
  asm volatile("mov.b32 %0, 0x41804180;" : "=r"(sixteens));
  // Where this lane finds its operands in a chunk (rows eight and sixteen further on lie as many rows further).
  const int own_key = key_of_row<DIM>(g), v_key[2] = {key_of_row<DIM>(2 * t), key_of_row<DIM>(2 * t + 1)};
  const int k_own = DIM == 128 ? piece_at<DIM>(own_key, t) : own_key * (DIM / 2) + t * 8;
  const int v_own[2] = {DIM == 128 ? piece_at<DIM>(v_key[0], g >> 1) + (g & 1) * 8 : v_key[0] * (DIM / 2) + g * 4,
                        DIM == 128 ? piece_at<DIM>(v_key[1], g >> 1) + (g & 1) * 8 : v_key[1] * (DIM / 2) + g * 4};
  pdl_wait();

  // ---- the chunks of every request (KV heads, blocks of columns and chunks of 32 keys), their running sum, this block's share ----
  auto span_of = [&](int r, int& first_key, int& n_rows) {      // chunks of a pair of request r
    const int t0 = p.q_start[r], n = p.q_start[r + 1] - t0;
    n_rows = 0;
    if (n <= 0 || (p.only_single && n > 1)) return 0;
    n_rows = n * p.per;
    const int last = min(p.positions[t0 + n - 1], p.reach - 1), begin = p.positions[t0];
    first_key = p.window > 0 ? max(0, begin - p.window + 1) / kChunk * kChunk : 0;
    return max(1, last < first_key ? 1 : (last - first_key) / kChunk + 1);       // (rows that see nothing are written too)
  };
  for (int r = threadIdx.x; r < p.n_requests; r += kThreads) {
    int first_key, n_rows;
    const int chunks = span_of(r, first_key, n_rows);
    cum_pairs[r + 1] = (n_rows + COLS - 1) / COLS * p.pages.g;
    cum[r + 1] = chunks;
    // (places behind the table have no page)
    if (n_rows > 0 && blockIdx.x == 0 && p.error && p.positions[p.q_start[r + 1] - 1] >= p.reach) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);
  }
  if (threadIdx.x == 0) cum[0] = cum_pairs[0] = 0;
  __syncthreads();
  if (warp == 0) {
    long long carry = 0;
    int carry_pairs = 0, most = 0;
    for (int r0 = 0; r0 < p.n_requests; r0 += 32) {
      const int r = r0 + lane;
      int pairs = r < p.n_requests ? cum_pairs[r + 1] : 0;
      long long v = r < p.n_requests ? cum[r + 1] : 0;
      most = max(most, (int)v);
      v *= pairs;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        const int w = __shfl_up_sync(0xffffffffu, pairs, o);
        if (lane >= o) { v += u; pairs += w; }
      }
      if (r < p.n_requests) { cum[r + 1] = carry + v; cum_pairs[r + 1] = carry_pairs + pairs; }
      carry += __shfl_sync(0xffffffffu, v, 31);
      carry_pairs += __shfl_sync(0xffffffffu, pairs, 31);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
      const Deal deal = carry > 0 ? choose_deal(p.slots, carry_pairs, most, carry) : Deal{0, 0};
      s_deal[0] = deal.pieces;
      s_deal[1] = deal.blocks;
    }
  }
  __syncthreads();
  const long long total = cum[p.n_requests];
  const int pieces = s_deal[0], blocks = s_deal[1];
  if ((int)blockIdx.x >= blocks) { pdl_launch_dependents(); return; }
  auto last_at_most = [&](auto* sums, auto value) {             // the request whose range of the running sum holds `value`
    int lo = 0, hi = p.n_requests - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sums[mid] <= value) lo = mid; else hi = mid - 1;
    }
    return lo;
  };
  auto share = [&](int b) { return (long long)b * total / blocks; };
  long long at, end;
  int req, first_block = 0, n_blocks = 1;                       // the blocks that hold the current pair
  if (pieces > 0) {
    const int pair = blockIdx.x / pieces, piece = blockIdx.x - pair * pieces;
    req = last_at_most(cum_pairs, pair);
    const int chunks = (int)((cum[req + 1] - cum[req]) / (cum_pairs[req + 1] - cum_pairs[req]));
    first_block = pair * pieces;
    n_blocks = min(pieces, chunks);
    if (piece >= n_blocks) { pdl_launch_dependents(); return; }
    at = cum[req] + (long long)(pair - cum_pairs[req]) * chunks;
    end = at + (long long)(piece + 1) * chunks / n_blocks;
    at += (long long)piece * chunks / n_blocks;
  } else {
    at = share(blockIdx.x);
    end = share(blockIdx.x + 1);
    req = last_at_most(cum, at);
  }

  for (bool first_of_block = true; at < end; first_of_block = false) {
    while (cum[req + 1] <= at) ++req;
    int first_key, n_rows;
    const int chunks = span_of(req, first_key, n_rows);
    const int col_blocks = (n_rows + COLS - 1) / COLS;
    const long long inside = at - cum[req];
    const int sub = (int)(inside / chunks), kvh = sub / col_blocks, column0 = (sub - kvh * col_blocks) * COLS;
    const int lo = (int)(inside - (long long)sub * chunks), hi = (int)min((long long)chunks, lo + (end - at));    // chunks [lo, hi) of the pair
    const long long first = at - lo;                            // its first chunk among all
    at += hi - lo;
    if (pieces == 0) {
      auto holder = [&](long long chunk) { return (int)(((chunk + 1) * blocks + total - 1) / total) - 1; };
      first_block = holder(first);
      n_blocks = holder(first + chunks - 1) - first_block + 1;
    }

    // ---- columns: the keys that each sees ----
    const int tok0 = p.q_start[req], score_row0 = p.only_single ? req : tok0;
    const int32_t* table_row = p.block_table + (size_t)req * p.table_width;
    int see_hi[NT][2], see_lo[NT][2], all_hi = 0x7fffffff, all_lo = 0, any_hi = -1, any_lo = 0x7fffffff;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int column = column0 + nt * 8 + 2 * t + e;
        see_hi[nt][e] = 0x7fffffff;
        see_lo[nt][e] = 0;
        if (column < n_rows) {
          see_hi[nt][e] = p.positions[tok0 + column / p.per];
          see_lo[nt][e] = p.window > 0 ? max(0, see_hi[nt][e] - p.window + 1) : 0;
          all_hi = min(all_hi, see_hi[nt][e]);
          all_lo = max(all_lo, see_lo[nt][e]);
          any_hi = max(any_hi, see_hi[nt][e]);
          any_lo = min(any_lo, see_lo[nt][e]);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, o));
      all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, o));
      any_hi = max(any_hi, __shfl_xor_sync(0xffffffffu, any_hi, o));
      any_lo = min(any_lo, __shfl_xor_sync(0xffffffffu, any_lo, o));
    }

    any_hi = min(any_hi, p.reach - 1);

    // Chunks of this warp that any column sees: one in kWarps.
    int c = lo + warp, c_end = hi;
    if (any_hi < 0) c_end = 0;
    else c_end = min(c_end, any_hi < first_key ? 0 : (any_hi - first_key) / kChunk + 1);
    if (any_lo > first_key) {
      const int skip = (any_lo - first_key) / kChunk;
      while (c < skip) c += kWarps;
    }
    // The pool's row of the chunk's first key (chunks inside pages) or of the lane's key, -1 without a page or for nobody's key.
    auto lookup = [&](int chunk) {
      const int key0 = first_key + chunk * kChunk, key = p.together == 2 ? key0 : key0 + lane;
      if (key > any_hi) return -1;
      const int index = p.pages.shift >= 0 ? key >> p.pages.shift : key / p.pages.page_size;
      const int page = index < p.table_width ? table_row[index] : -1;
      if ((unsigned)page >= (unsigned)p.pages.num_pages) {
        if ((p.together == 2 ? key0 + kChunk - 1 : key) >= any_lo && p.error) atomicOr(p.error, YALIS_FLAG_BAD_PAGE);
        return -1;
      }
      return (page * p.pages.g + kvh) * p.pages.page_size + (key - index * p.pages.page_size);
    };
    // Rows that are not there are left as they are: their word says so.
    auto ask = [&](int chunk, int stage, int row) {
      Stage<DIM>& st = ring[stage];
      const uint32_t k_at = smem_u32(st.k), v_at = smem_u32(st.v);
      if (p.together == 2) {                     // (rows behind the last key are copied too, here and below)
        if (row >= 0) {
          const uint32_t own = piece_at<DIM>(lane / PIECES, lane % PIECES);
          const size_t byte = (size_t)row * (DIM / 2) + lane * 16;
          const unsigned char *k_from = reinterpret_cast<const unsigned char*>(p.pages.k) + byte, *v_from = reinterpret_cast<const unsigned char*>(p.pages.v) + byte;
#pragma unroll
          for (int i = 0; i < COPIES; ++i) {
            copy16(k_at + own + i * 512, k_from + i * 512);
            copy16(v_at + own + i * 512, v_from + i * 512);
          }
          row += lane;
        }
        if (first_key + chunk * kChunk + lane > any_hi) row = -1;
      } else if (p.together) {                   // a lane's pieces are neighbours of the group's first row
        const uint32_t own = piece_at<DIM>(lane / PIECES, lane % PIECES);
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
          const int from = __shfl_sync(0xffffffffu, row, i * (32 / PIECES));
          if (from >= 0) {
            const size_t byte = (size_t)from * (DIM / 2) + lane * 16;
            copy16(k_at + own + i * 512, reinterpret_cast<const unsigned char*>(p.pages.k) + byte);
            copy16(v_at + own + i * 512, reinterpret_cast<const unsigned char*>(p.pages.v) + byte);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
          const int r = i * (32 / PIECES) + lane / PIECES, piece = lane % PIECES;
          const int from = __shfl_sync(0xffffffffu, row, r);
          if (from >= 0) {
            const size_t byte = (size_t)from * (DIM / 2) + piece * 16;
            copy16(k_at + piece_at<DIM>(r, piece), reinterpret_cast<const unsigned char*>(p.pages.k) + byte);
            copy16(v_at + piece_at<DIM>(r, piece), reinterpret_cast<const unsigned char*>(p.pages.v) + byte);
          }
        }
      }
      if (row >= 0) copy4(smem_u32(&st.words[lane]), p.pages.words + row);
      else st.words[lane] = 0u;
    };
    int row = -1;
    if (c < c_end) ask(c, 0, lookup(c));
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (c + kWarps < c_end) row = lookup(c + kWarps);

    // ---- queries in registers as the products' right operand, while the first copies are under way ----
    // HALF: in float16, by a power of two (unit takes it out again) so high that a column's largest is 2^11 to 2^12: no bit is lost of
    // anything above 2^-28 of it.  The pairs whose codes lie in the lowest bits go in sixteenfold.
    uint32_t qf[NT][2 * W][2][PARTS];
    float q_sum[NT][2], unit[NT][2];             // sum(q) of the columns 2t, 2t + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = column0 + nt * 8 + g;
      const bool real = row < n_rows;
      const int token = tok0 + (real ? row / p.per : 0), head = kvh * p.per + (real ? row % p.per : 0);
      const T* src = static_cast<const T*>(p.q) + (long long)token * p.q_stride + (long long)head * DIM + t * (DIM / 4);
      float x[W][8], own = 0.f, own_unit = 1.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (!real) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[w][i] = 0.f;
        } else if (p.q_vector) {
          const float4 a = load4_f32(src + 8 * w), b = load4_f32(src + 8 * w + 4);
          x[w][0] = a.x; x[w][1] = a.y; x[w][2] = a.z; x[w][3] = a.w;
          x[w][4] = b.x; x[w][5] = b.y; x[w][6] = b.z; x[w][7] = b.w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[w][i] = to_f32<T>(src[8 * w + i]);
        }
      }
      float scale = 1.f;
      if constexpr (HALF) {
        uint32_t most = 0u;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[w][i]) & 0x7FFFFFFFu);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2)) >> 23;
        const uint32_t up = min(254u, 265u - most);
        const bool fits = most < 246u;           // (nothing from 2^119 on is computed with)
        scale = fits ? __uint_as_float(up << 23) : NAN;
        own_unit = fits ? __uint_as_float((274u - up) << 23) : 1.f;             // 2^20 / scale: codes are 2^-24 and 2^-20 of their numbers
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (HALF) {
            const float a = x[w][i] * scale, b = x[w][i + 4] * scale;
            own += a + b;
            qf[nt][2 * w + (i >> 1)][i & 1][0] = i & 1 ? pair_f16(a, b) : pair_f16(16.f * a, 16.f * b);
          } else {
            parts_of<PARTS>(x[w][i], x[w][i + 4], qf[nt][2 * w + (i >> 1)][i & 1]);
            own += x[w][i] + x[w][i + 4];
          }
        }
      }
      if constexpr (HALF) own *= 9.5367431640625e-7f;          // 2^-20: in the products' unit
      own += __shfl_xor_sync(0xffffffffu, own, 1);
      own += __shfl_xor_sync(0xffffffffu, own, 2);             // column g, in its four lanes
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        q_sum[nt][e] = __shfl_sync(0xffffffffu, own, (2 * t + e) * 4);
        unit[nt][e] = HALF ? __shfl_sync(0xffffffffu, own_unit, (2 * t + e) * 4) : 1.f;
      }
    }

    // Scores are taken relative to base; one above limit (HALF: with the value's step, both in powers of two) moves it.
    float base[NT][2], limit[NT][2], l[NT][2], acc[NT][MT][4], acc_z[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      base[nt][0] = base[nt][1] = l[nt][0] = l[nt][1] = 0.f;
      limit[nt][0] = limit[nt][1] = kUnset;
      acc_z[nt][0] = acc_z[nt][1] = acc_z[nt][2] = acc_z[nt][3] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
    }

    for (int stage = 0; c < c_end; c += kWarps, stage ^= 1) {
      if (c + kWarps < c_end) ask(c + kWarps, stage ^ 1, row);
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (c + 2 * kWarps < c_end) row = lookup(c + 2 * kWarps);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      const Stage<DIM>& st = ring[stage];
      const int key0 = first_key + c * kChunk;
      float4 own = terms_of(st.words[lane], p.scale_log2);
      if constexpr (HALF) {
        own.y -= 16.f;                           // (no sixteens in the keys' codes)
        // log2 of the value's step.  (Where that is no number its rows have no results, but their weights' sums are as ever.)
        height[lane] = own.z <= 3.4e38f ? fmaxf((float)((int)(__float_as_uint(own.z) >> 23) - 127), kSmall) : kSmall;
        own.w = __uint_as_float(st.words[lane] >> 16 & 15u);   // the value's zero times 2^-24 in float16
      }
      terms[lane] = own;
      __syncwarp();

      // ---- products with 32 keys ----
      float sc[NT][2][4];
      float4 term[2][2];
      float rise[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        term[half][0] = terms[own_key + half * 16];
        term[half][1] = terms[own_key + half * 16 + 8];
        if constexpr (HALF) {
          rise[half][0] = height[own_key + half * 16];
          rise[half][1] = height[own_key + half * 16 + 8];
        }
        uint32_t wa[W], wb[W];
        const unsigned char* from = st.k + k_own + half * 16 * (DIM / 2);
        if constexpr (DIM == 128) {
          *reinterpret_cast<uint4*>(wa) = *reinterpret_cast<const uint4*>(from);
          *reinterpret_cast<uint4*>(wb) = *reinterpret_cast<const uint4*>(from + 8 * (DIM / 2));
        } else {
          *reinterpret_cast<uint2*>(wa) = *reinterpret_cast<const uint2*>(from);
          *reinterpret_cast<uint2*>(wb) = *reinterpret_cast<const uint2*>(from + 8 * (DIM / 2));
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][half][0] = sc[nt][half][1] = sc[nt][half][2] = sc[nt][half][3] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint32_t lo[4], hi[4];
          if constexpr (HALF) {                  // as they lie: c in the lowest bits is c 2^-24 in float16, c in the next c 2^-20
            const uint32_t wa8 = wa[w] >> 8, wb8 = wb[w] >> 8;
            lo[0] = wa[w] & 0x000F000Fu; lo[1] = wb[w] & 0x000F000Fu; lo[2] = wa[w] & 0x00F000F0u; lo[3] = wb[w] & 0x00F000F0u;
            hi[0] = wa8 & 0x000F000Fu; hi[1] = wb8 & 0x000F000Fu; hi[2] = wa8 & 0x00F000F0u; hi[3] = wb8 & 0x00F000F0u;
          } else {
            lo[0] = code_pair<0>(wa[w], sixteens); lo[1] = code_pair<0>(wb[w], sixteens); lo[2] = code_pair<1>(wa[w], sixteens); lo[3] = code_pair<1>(wb[w], sixteens);
            hi[0] = code_pair<2>(wa[w], sixteens); hi[1] = code_pair<2>(wb[w], sixteens); hi[2] = code_pair<3>(wa[w], sixteens); hi[3] = code_pair<3>(wb[w], sixteens);
            const uint32_t za = __byte_perm(__float_as_uint(term[half][0].y), 0, 0x3232), zb = __byte_perm(__float_as_uint(term[half][1].y), 0, 0x3232);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              lo[i] = minus(lo[i], i & 1 ? zb : za);
              hi[i] = minus(hi[i], i & 1 ? zb : za);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = PARTS - 1; i >= 0; --i) {
              if constexpr (HALF) {
                mma_f16(sc[nt][half], lo, qf[nt][2 * w][0][i], qf[nt][2 * w][1][i]);
                mma_f16(sc[nt][half], hi, qf[nt][2 * w + 1][0][i], qf[nt][2 * w + 1][1][i]);
              } else {
                mma_bf16(sc[nt][half], lo, qf[nt][2 * w][0][i], qf[nt][2 * w][1][i]);
                mma_bf16(sc[nt][half], hi, qf[nt][2 * w + 1][0][i], qf[nt][2 * w + 1][1][i]);
              }
            }
          }
        }
      }
      // ---- softmax: scores in powers of two, less the maximum in use ----
      if constexpr (HALF) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[nt][half][i] = fmaf(-term[half][i >> 1].y, q_sum[nt][i & 1], sc[nt][half][i]);
      }
      auto weigh = [&](auto mask) {              // sc: products in, weights times the values' steps out
        constexpr bool MASK = decltype(mask)::value;
        if constexpr (SCORES) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int column = column0 + nt * 8 + 2 * t + x;
              if (column >= n_rows) continue;
              float* to = p.scores + ((size_t)(score_row0 + column / p.per) * p.nh + kvh * p.per + column % p.per) * p.score_stride + key0;
#pragma unroll
              for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int j = half * 16 + own_key + 8 * e;
                  if ((!MASK || key0 + j <= see_hi[nt][x]) && key0 + j < p.score_stride)
                    to[j] = MASK && term[half][e].z == 0.f ? -INFINITY : term[half][e].x * unit[nt][x] * sc[nt][half][2 * e + x];
                }
            }
        }
        float most[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) most[nt][0] = most[nt][1] = -INFINITY;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float& v = sc[nt][half][i];
              v = fmaf(HALF ? term[half][i >> 1].x * unit[nt][i & 1] : term[half][i >> 1].x, v, -base[nt][i & 1]);
              if constexpr (MASK) {
                const int key = key0 + half * 16 + own_key + 8 * (i >> 1);
                if (!(key <= see_hi[nt][i & 1] && key >= see_lo[nt][i & 1] && term[half][i >> 1].z != 0.f)) v = -INFINITY;
              }
              most[nt][i & 1] = fmaxf(most[nt][i & 1], HALF ? v + rise[half][i >> 1] : v);
            }
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) grow |= most[nt][0] > limit[nt][0] || most[nt][1] > limit[nt][1];
        if (__any_sync(0xffffffffu, grow)) {       // seldom after the first chunks: the base moves, what was summed is rescaled
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float keep[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float top = most[nt][x];
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
              constexpr float kTo = HALF ? kTarget : 0.f;
              float up = fmaxf(top - kTo, 0.f);
              keep[x] = exp2_fast(-up);
              if (limit[nt][x] == kUnset) {        // nothing summed yet: the first maximum, wherever it lies
                up = top == -INFINITY ? 0.f : top - kTo;
                limit[nt][x] = top == -INFINITY ? kUnset : kTo + kLazy;
                keep[x] = 1.f;
              }
              base[nt][x] += up;
              l[nt][x] *= keep[x];
#pragma unroll
              for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int e = 0; e < 2; ++e) sc[nt][half][2 * e + x] -= up;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              acc[nt][i][0] *= keep[0]; acc[nt][i][1] *= keep[1];
              acc[nt][i][2] *= keep[0]; acc[nt][i][3] *= keep[1];
            }
            acc_z[nt][0] *= keep[0]; acc_z[nt][1] *= keep[1];
            acc_z[nt][2] *= keep[0]; acc_z[nt][3] *= keep[1];
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = sc[nt][half][i], e = PARTS == 1 ? exp2_fast(v) : exp2f(v);
              l[nt][i & 1] += e;
              sc[nt][half][i] = MASK && v == -INFINITY ? 0.f : e * term[half][i >> 1].z;         // a row that is not seen may hold anything
            }
      };
      // (a key without a page is hidden from every column)
      if (__any_sync(0xffffffffu, key0 + kChunk - 1 > all_hi || key0 < all_lo || own.z == 0.f)) weigh(std::true_type());
      else weigh(std::false_type());
      uint32_t wf[NT][2][2][PARTS];              // [half][keys g, g + 8 of the half]: the weights as the second product's operand
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (HALF) {
              wf[nt][half][e][0] = transposed(pair_f16(sc[nt][half][2 * e], sc[nt][half][2 * e + 1]));
            } else {
              uint32_t part[PARTS];
              parts_of<PARTS>(sc[nt][half][2 * e], sc[nt][half][2 * e + 1], part);
#pragma unroll
              for (int i = 0; i < PARTS; ++i) wf[nt][half][e][i] = transposed(part[i]);
            }
          }
      // ---- output ----
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t vw[4][U];
        float z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {            // keys of rows 2t, 2t + 1, 2t + 8, 2t + 9
          z[i] = terms[v_key[i & 1] + half * 16 + (i & 2) * 4].w;
          const unsigned char* from = st.v + v_own[i & 1] + (half * 16 + (i & 2) * 4) * (DIM / 2);
          if constexpr (DIM == 128) {
            const uint2 two = *reinterpret_cast<const uint2*>(from);
            vw[i][0] = two.x;
            vw[i][U - 1] = two.y;
          } else {
            vw[i][0] = *reinterpret_cast<const uint32_t*>(from);
          }
        }
        if constexpr (HALF) {
          const uint32_t z01 = __byte_perm(__float_as_uint(z[0]), __float_as_uint(z[1]), 0x5410), z23 = __byte_perm(__float_as_uint(z[2]), __float_as_uint(z[3]), 0x5410);
          const uint32_t zeros[4] = {z01, z01, z23, z23};      // every row of a tile of its own
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(acc_z[nt], zeros, wf[nt][half][0][0], wf[nt][half][1][0]);
#pragma unroll
          for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t a = __byte_perm(vw[0][u], vw[1][u], h ? 0x7632 : 0x5410), b = __byte_perm(vw[2][u], vw[3][u], h ? 0x7632 : 0x5410);
              const uint32_t a8 = a >> 8, b8 = b >> 8;
              const uint32_t f0[4] = {a & 0x000F000Fu, a & 0x00F000F0u, b & 0x000F000Fu, b & 0x00F000F0u};
              const uint32_t f1[4] = {a8 & 0x000F000Fu, a8 & 0x00F000F0u, b8 & 0x000F000Fu, b8 & 0x00F000F0u};
              const int tile = 4 * u + 2 * h;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_f16(acc[nt][tile], f0, wf[nt][half][0][0], wf[nt][half][1][0]);
                mma_f16(acc[nt][tile + 1], f1, wf[nt][half][0][0], wf[nt][half][1][0]);
              }
            }
          }
        } else {
          const uint32_t z01 = __byte_perm(__float_as_uint(z[0]), __float_as_uint(z[1]), 0x7632);
          const uint32_t z23 = __byte_perm(__float_as_uint(z[2]), __float_as_uint(z[3]), 0x7632);
#pragma unroll
          for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t a = __byte_perm(vw[0][u], vw[1][u], h ? 0x7632 : 0x5410), b = __byte_perm(vw[2][u], vw[3][u], h ? 0x7632 : 0x5410);
              const uint32_t f0[4] = {minus(code_pair<0>(a, sixteens), z01), minus(code_pair<1>(a, sixteens), z01), minus(code_pair<0>(b, sixteens), z23),
                                      minus(code_pair<1>(b, sixteens), z23)};
              const uint32_t f1[4] = {minus(code_pair<2>(a, sixteens), z01), minus(code_pair<3>(a, sixteens), z01), minus(code_pair<2>(b, sixteens), z23),
                                      minus(code_pair<3>(b, sixteens), z23)};
              const int tile = 4 * u + 2 * h;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {  // added to the running output by float32 additions: the tensor cores cut sums off
                float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = PARTS - 1; i >= 0; --i) {
                  mma_bf16(d0, f0, wf[nt][half][0][i], wf[nt][half][1][i]);
                  mma_bf16(d1, f1, wf[nt][half][0][i], wf[nt][half][1][i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  acc[nt][tile][i] += d0[i];
                  acc[nt][tile + 1][i] += d1[i];
                }
              }
            }
          }
        }
      }
      __syncwarp();                              // the stage is read: the next round may fill it
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (at >= end) pdl_launch_dependents();      // this block's last tile is there

    if constexpr (HALF) {                        // codes and zeros were taken by 2^24 too small, those of odd elements by 2^20
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          acc[nt][i][0] = (acc[nt][i][0] - acc_z[nt][0]) * 16777216.f;
          acc[nt][i][1] = (acc[nt][i][1] - acc_z[nt][1]) * 16777216.f;
          acc[nt][i][2] = (acc[nt][i][2] - 16.f * acc_z[nt][2]) * 1048576.f;
          acc[nt][i][3] = (acc[nt][i][3] - 16.f * acc_z[nt][3]) * 1048576.f;
        }
    }
    // A sum of weights on a base `by` higher.  HALF: bases may lie further apart than float32's powers of two, by the values' steps.
    auto moved = [](float sum, float by) {
      if constexpr (HALF) {
        const float half = exp2f(0.5f * by);
        return sum * half * half;
      } else {
        return sum * exp2f(by);
      }
    };
    // ---- the four warps' results together ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], o);
    constexpr int OWN = MT / kWarps;             // tiles of each column block that a warp finishes: its lanes' elements are neighbours
    float4 sum[NT][OWN];
    float top[NT][2], norm[NT][2];
    auto together = [&]() {                      // base, l, acc of every warp -> top, norm, sum
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (g == 0) *reinterpret_cast<float2*>(merge_ml + (warp * COLS + nt * 8 + 2 * t + x) * 2) = make_float2(limit[nt][x] == kUnset ? kNone : base[nt][x], l[nt][x]);
#pragma unroll
        for (int i = 0; i < MT; ++i)
          merge_o[(warp * NT * MT + nt * MT + i) * 32 + lane] = make_float4(acc[nt][i][0], acc[nt][i][1], acc[nt][i][2], acc[nt][i][3]);
      }
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float2 ml[kWarps][2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          top[nt][x] = kNone;
          norm[nt][x] = 0.f;
#pragma unroll
          for (int k = 0; k < kWarps; ++k) {
            ml[k][x] = *reinterpret_cast<const float2*>(merge_ml + (k * COLS + nt * 8 + 2 * t + x) * 2);
            top[nt][x] = fmaxf(top[nt][x], ml[k][x].x);
          }
        }
#pragma unroll
        for (int i = 0; i < OWN; ++i) sum[nt][i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          const float f0 = exp2f(ml[k][0].x - top[nt][0]), f1 = exp2f(ml[k][1].x - top[nt][1]);
          norm[nt][0] += moved(ml[k][0].y, ml[k][0].x - top[nt][0]);
          norm[nt][1] += moved(ml[k][1].y, ml[k][1].x - top[nt][1]);
#pragma unroll
          for (int i = 0; i < OWN; ++i) {
            const float4 v = merge_o[(k * NT * MT + nt * MT + warp * OWN + i) * 32 + lane];
            sum[nt][i].x += v.x * f0; sum[nt][i].z += v.z * f0;
            sum[nt][i].y += v.y * f1; sum[nt][i].w += v.w * f1;
          }
        }
      }
    };
    together();
    bool finish = n_blocks == 1;
    if (!finish) {
      // A block's share begins inside one pair and ends inside another at most: two places of its own.
      auto place = [&](int b, bool its_first) { return p.part + ((size_t)b * 2 + (its_first ? 0 : 1)) * PART_FLOATS; };
      float* mine = place(blockIdx.x, first_of_block);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < OWN; ++i) reinterpret_cast<float4*>(mine)[(nt * MT + warp * OWN + i) * 32 + lane] = sum[nt][i];
        if (warp == 0 && g == 0)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            *reinterpret_cast<float2*>(mine + NT * MT * 128 + (nt * 8 + 2 * t + x) * 2) = make_float2(top[nt][x], norm[nt][x]);
      }
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {                    // (one pair at most goes on from a block to the next: the first block's number is its counter)
        const bool last = atomicAdd(p.tickets + first_block, 1) == n_blocks - 1;
        if (last) p.tickets[first_block] = 0;
        *s_last = last;
      }
      __syncthreads();
      finish = *s_last != 0;
      if (finish) {                              // the blocks' results, every fourth a warp's, then the warps' as before
        __threadfence();
        const bool begins = pieces > 0 || share(first_block) >= first;      // whether the pair is the first of its first block
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          base[nt][0] = base[nt][1] = kNone;
          limit[nt][0] = limit[nt][1] = kLazy;
          l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
        }
        for (int k = warp; k < n_blocks; k += kWarps) {
          const float* from = place(first_block + k, k > 0 || begins);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float4 v[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) v[i] = __ldcg(reinterpret_cast<const float4*>(from) + (nt * MT + i) * 32 + lane);
            float was[2], is[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(from + NT * MT * 128 + (nt * 8 + 2 * t + x) * 2));
              const float next = fmaxf(base[nt][x], ml.x);
              was[x] = exp2f(base[nt][x] - next);
              is[x] = exp2f(ml.x - next);
              l[nt][x] = moved(l[nt][x], base[nt][x] - next) + moved(ml.y, ml.x - next);
              base[nt][x] = next;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              acc[nt][i][0] = acc[nt][i][0] * was[0] + v[i].x * is[0];
              acc[nt][i][1] = acc[nt][i][1] * was[1] + v[i].y * is[1];
              acc[nt][i][2] = acc[nt][i][2] * was[0] + v[i].z * is[0];
              acc[nt][i][3] = acc[nt][i][3] * was[1] + v[i].w * is[1];
            }
          }
        }
        together();
      }
    }
    if (finish) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int column = column0 + nt * 8 + 2 * t + x;
          if (column >= n_rows) continue;
          const int token = tok0 + column / p.per, head = kvh * p.per + column % p.per;
          const float inv = norm[nt][x] == 0.f ? 0.f : 1.f / norm[nt][x];
          T* dst = static_cast<T*>(p.out) + (long long)token * p.out_stride + (long long)head * DIM + g * (DIM / 8) + warp * OWN * 2;
#pragma unroll
          for (int i = 0; i < OWN; ++i) {
            const float a = x ? sum[nt][i].y : sum[nt][i].x, b = x ? sum[nt][i].w : sum[nt][i].z;
            dst[2 * i] = from_f32<T>(a * inv);
            dst[2 * i + 1] = from_f32<T>(b * inv);
          }
          if (p.lse2 && warp == 0 && g == 0) p.lse2[(size_t)token * p.nh + head] = top[nt][x] + log2f(norm[nt][x]);
        }
      }
    }
    __syncthreads();                             // the merge's memory is free again
  }
}

template <typename T, int DIM, int NT, int PARTS, bool SCORES>
int launch_mma_as(const MmaParams& p, int grid, cudaStream_t stream) {
  constexpr int MT = DIM / 16;
  const size_t smem = sizeof(Stage<DIM>) * kStages * kWarps + kWarps * kChunk * 20 + (size_t)kWarps * NT * MT * 512 + (size_t)kWarps * 8 * NT * 8 + 16 +
                      (size_t)(p.n_requests + 1) * 12;
  auto* kernel = packed_attention_mma_kernel<T, DIM, NT, PARTS, SCORES>;
  static int configured[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return YALIS_ERR_LAUNCH;
  if (smem > 200 * 1024) return YALIS_ERR_SHAPE;
  if (dev < 0 || dev >= 64 || configured[dev] < (int)smem) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return YALIS_ERR_LAUNCH;
    if (dev >= 0 && dev < 64) configured[dev] = (int)smem;
  }
  return yalis_launch(kernel, dim3(grid), dim3(kThreads), smem, stream, p);
}

template <typename T, int DIM, int NT, int PARTS>
int launch_mma(const MmaParams& p, int grid, cudaStream_t stream) {
  return p.scores ? launch_mma_as<T, DIM, NT, PARTS, true>(p, grid, stream) : launch_mma_as<T, DIM, NT, PARTS, false>(p, grid, stream);
}

}  // namespace

// Blocks of the launch (the same for every step of these shapes), and the floats of scratch memory that it needs.
YALIS_API int yalis_packed_attention_mma_blocks(int dtype, int dim, int columns) {
  return yalis_sm_count() * (dtype == YALIS_BF16 && columns <= 8 ? 4 : 2);
}
YALIS_API long long yalis_packed_attention_mma_scratch_floats(int blocks, int dim, int columns) {
  const int nt = columns <= 8 ? 1 : 2;
  return (long long)blocks * 2 * (nt * (dim / 16) * 128 + 16 * nt);
}

// `columns`: 8 or 16, the query rows of a pair (float32: 8); `max_rows`: the most that a request has for a KV head.  `blocks`, scratch
// memory and as many tickets: see above.
YALIS_API int yalis_packed_attention_mma(const void* q, long long q_stride, int dtype, void* out, long long out_stride, void* k_codes,
                                         void* v_codes, void* words, int num_pages, int page_size, int g, int dim, const int32_t* positions,
                                         const int32_t* q_start, const int32_t* block_table, int table_width, int n_requests, int nh,
                                         int columns, int q_vector, int only_single, float scale, int window, float* lse2, float* scores,
                                         long long score_stride, int max_rows, int blocks, float* scratch, int32_t* tickets, int32_t* error, cudaStream_t stream) {
  if ((dim != 64 && dim != 128) || nh % g || n_requests > 4096 || blocks < 1) return YALIS_ERR_SHAPE;
  if (n_requests <= 0) return YALIS_OK;
  MmaParams p = {};
  p.q = q; p.q_stride = q_stride; p.out = out; p.out_stride = out_stride;
  p.positions = positions; p.q_start = q_start; p.block_table = block_table; p.table_width = table_width;
  p.n_requests = n_requests; p.nh = nh; p.per = nh / g; p.window = window; p.q_vector = q_vector; p.only_single = only_single;
  p.together = page_size % kChunk == 0 ? 2 : page_size % (1024 / dim) == 0 ? 1 : 0;
  p.slots = blocks;
  p.reach = (int)min((long long)table_width * page_size, 0x7fffffffll);
  const long long pairs = (long long)n_requests * g * ((max_rows + columns - 1) / columns), grid = pairs > blocks ? pairs : blocks;
  if (grid > 0x7fffffffll) return YALIS_ERR_SHAPE;
  p.scale_log2 = scale * 1.4426950408889634f; p.lse2 = lse2; p.scores = scores; p.score_stride = score_stride; p.part = scratch; p.tickets = tickets; p.error = error;
  p.pages = packed_pages(k_codes, v_codes, words, num_pages, page_size, g, dim);
  if (dtype == YALIS_BF16) {
    if (columns == 8) return dim == 64 ? launch_mma<__nv_bfloat16, 64, 1, 1>(p, (int)grid, stream) : launch_mma<__nv_bfloat16, 128, 1, 1>(p, (int)grid, stream);
    if (columns == 16) return dim == 64 ? launch_mma<__nv_bfloat16, 64, 2, 1>(p, (int)grid, stream) : launch_mma<__nv_bfloat16, 128, 2, 1>(p, (int)grid, stream);
  }
  if (dtype == YALIS_F32 && columns == 8)
    return dim == 64 ? launch_mma<float, 64, 1, 3>(p, (int)grid, stream) : launch_mma<float, 128, 1, 3>(p, (int)grid, stream);
  return YALIS_ERR_DTYPE;
}

YALIS_SLOTS(yalis_packed_attention_mma)
