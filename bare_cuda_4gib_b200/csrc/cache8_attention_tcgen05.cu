// Softmax attention of prompt portions over a cache of e4m3 codes (cache8.cuh) on the Blackwell tensor cores: what
// attention_tcgen05.cu is to a bfloat16 cache, for requests with more than 16 packed rows (tokens x query heads of one key/value
// head).  Nothing of cuongvng/bare-cuda-4gib's [heads, T, keys] score buffer exists (engine/kernels/attention_qk.cu:49-68,
// softmax.cu:28-42, attention_av.cu:24-44).
//
//   s[k] = scale * 2^e_K(k) * (q . K_k)     p = softmax over the visible k     out = sum_k p[k] 2^e_V(k) V_k
//
// One thread block = two tiles of 128 packed rows of one request and one key/value head, which share every key and value block of 128
// positions.  Warps:
//   loader (1)     copies a key block's codes, as they lie in the request's pages, into a ring of their own with TMA (one tensor map over the cache's
//                  pool, a box per piece of a page), and splits the block's scales into 2^e (the largest, which the softmax gets) and what is
//                  left for 16 positions, at most one, which the converters get;
//   converters (4) write a tile's codes as halves, times what is left of their scale (exact down to 2^-15), into 128-byte-swizzled shared
//                  memory.  Halves hold e4m3 exactly and one instruction converts two codes.  Key tiles and value tiles go through ONE ring
//                  of slots in the order K(0) V(0) K(1) ...;
//   MMA issuers (2) S_g = Q_g K^T (M 128, N 128, K head size) into tile g's S columns of tensor memory, and
//                  O_g (+)= P_g V with P_g as the operand in tensor memory and V as it lies ([key][channel], MN-major), in two halves of 64
//                  keys, each as soon as its half of P is there: P never goes through shared memory, whose bandwidth
//                  is what a block with P there is bound by (K and V tiles, two Q tiles and two P tiles a key block);
//   softmax (8)    a group of four warps per tile, one thread per row.  First it stages Q_g as halves (times a power of two of
//                  the row's own).  Then, per key block: read the row of S, 64 columns at a time, mask, running maximum and sum in
//                  float32 (base 2), write P as halves back into tensor memory.
// A weight goes into P together with the scale of its block's values: P = 2^(s + e_V - m) with m the running maximum of s + e_V, while the sum
// takes P 2^-e_V.  So a half of P is relative to what the row's keys can add to its output, and O needs no factor of its own.
// m follows the true maximum only when that has grown by more than 2^8 (a half reaches 2^15), so O is rescaled rarely.
// A half of P takes the columns of the scores it was made of (S 2 x 128, O 2 x head size columns of the 512), and the next key block's half of S is
// issued when P has been read, while the softmax is at the other half: it waits for no product.
// Few tiles (a question behind a long text): the key blocks are split among the blocks of a cluster, each with a softmax of its own; their
// states are merged in index order through distributed shared memory.
// A NaN scale (a block that was given a NaN) makes keys NaN, hence the scores of the rows that see them; hidden scores are replaced, not
// multiplied, and values are finite always.  Values behind the request's last key are written as zeros.
// Every mbarrier wait is bounded: on a timeout the thread sets the error word, all roles leave their loops, tensor memory is
// released and the block returns.
// One B200: a prompt of 2,048 tokens (32 / 4 heads of 64) 44.2 us, 2,048 tokens behind 2,048 (32 heads of 128) 127 us, 61 tokens behind 3,001
// (32 / 8 heads of 128) 23.5 us.

#include "cache8.cuh"

#include <cuda.h>
#include <cuda_fp16.h>
#include <string.h>

#ifndef HEAD_DIM
#define HEAD_DIM 64
#endif

namespace {

constexpr int D = HEAD_DIM;
static_assert(D == 64 || D == 128, "the tcgen05 attention kernel is built for head sizes 64 and 128");
constexpr int KA = D / 64;       // 64-wide sub-tiles ("atoms") along the head dimension
constexpr int BM = 128;          // packed rows per tile (one softmax group)
constexpr int TILES = 2;         // tiles per block: both read every converted key and value tile
constexpr int BLOCK_ROWS = TILES * BM;
constexpr int BN = 128;          // keys per block
constexpr int SUB = 128 * 128;   // bytes of a [128 rows x 64 halves] swizzled sub-tile
constexpr int Q_BYTES = KA * SUB;        // one tile's queries
constexpr int TILE_BYTES = KA * SUB;     // one key tile or one value tile
constexpr int RAW_BYTES = BN * D;        // one key tile or one value tile as codes
constexpr int SLOTS = HEAD_DIM == 64 ? 6 : 3, RAW_SLOTS = HEAD_DIM == 64 ? 6 : 4;   // tiles in flight, as halves and as codes (what shared memory allows)
constexpr int SOFTMAX_THREADS = 128 * TILES, CONVERT_THREADS = 128;
constexpr int CONVERT_WARP = SOFTMAX_THREADS / 32, MMA_WARP = CONVERT_WARP + CONVERT_THREADS / 32, LOADER_WARP = MMA_WARP + TILES;
constexpr int NUM_THREADS = (LOADER_WARP + 1) * 32;   // warps 0-7 softmax, 8-11 converters, 12 and 13 MMA (one a tile), 14 loader
constexpr int GROUP_THREADS = 128;
constexpr int S_PIECE = 64;      // columns of S a softmax thread holds in registers at a time
constexpr int TMEM_COLS = 512, O_COL = TILES * BN;
constexpr unsigned long long WAIT_LIMIT_NS = 1000000000ull;
constexpr float RESCALE_STEP = 8.0f;
constexpr int CHUNKS = D / 16;              // 16-byte chunks of a key's codes; also how many of them a converter thread takes of a tile
constexpr int BLOCKS = BN / SCALE_TOKENS;   // scale blocks of a key block
constexpr int EXPONENTS = 16;               // key blocks whose exponents are kept (more than can be in flight)
constexpr int STATE = D + 4;                // floats of a row's state in a merge: D sums, the maximum, the sum
constexpr size_t TILES_BYTES = (size_t)TILES * Q_BYTES + (size_t)SLOTS * TILE_BYTES + (size_t)RAW_SLOTS * RAW_BYTES;
static_assert((size_t)BLOCK_ROWS * STATE * 4 <= TILES_BYTES, "the states of a merge lie over the tiles");
constexpr size_t SMEM_BYTES = TILES_BYTES + 768;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ unsigned long long global_timer() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long start = global_timer();
  for (unsigned spins = 0;; ++spins) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((spins & 63u) == 63u) {
      if (*abort_flag) return false;
      if (global_timer() - start > WAIT_LIMIT_NS) return false;
    }
  }
}

// Byte offset of the 16-byte chunk `chunk` (0..7) of row `row` inside a [rows x 64 bf16] sub-tile
// with the 128-byte swizzle: rows are 128 bytes, groups of 8 rows are 1024 bytes, and the chunk
// index is XORed with the row's index inside its group.
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
  return (uint32_t)((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4));
}

__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
}
// Byte offset of chunk `chunk` of row `row` in a tile of codes as TMA writes it: 128-byte swizzle for rows of 128 bytes, 64-byte swizzle
// for rows of 64.
__device__ __forceinline__ uint32_t raw_swizzled(int row, int chunk) {
  return (uint32_t)(row * D + ((D == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3)) << 4));
}

// Shared-memory matrix descriptor, 128-byte swizzle, 1024 bytes between 8-row groups.
__device__ __forceinline__ uint64_t smem_desc_sw128(uint32_t addr, uint32_t leading = 16) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(leading >> 4) << 16;      // MN-major operands: bytes from one 64-wide sub-tile to the next
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// float32 accumulator, half operands, A K-major; B K-major or (b_mn = 1) MN-major.
__host__ __device__ constexpr uint32_t instr_desc(int m, int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// The A operand in tensor memory: lane = row, 32-bit column c = its elements 2 c and 2 c + 1.
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tmem_load32_nowait(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Two float32 numbers in one register pair, and one instruction for both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpair(uint64_t a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Four codes as four halves.
__device__ __forceinline__ void halves(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// 2^-d twice as a half (zero where a half has no such number).
__device__ __forceinline__ uint32_t half_power(int d) {
  const uint32_t h = d <= 14 ? (uint32_t)(15 - d) << 10 : d <= 24 ? 1u << (24 - d) : 0u;
  return h | (h << 16);
}
__device__ __forceinline__ uint32_t peer_smem(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ float4 load_peer4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

struct AttnArgs {
  const __nv_bfloat16* q;      // [tokens, q_heads, D]
  __nv_bfloat16* out;          // [tokens, q_heads * D]
  Cache8 cache;
  long long page_rows, k_row0, v_row0;   // the pool seen as rows of D codes: row = page * page_rows + k_row0 (or v_row0) + kv head * page_tokens + ...
  int box_rows;                // rows of the tensor map's box: divides the page size and BN
  StepLists lists;
  int q_heads;
  float scale_log2;
  int window;
  AttentionExtras extras;
  int* error_word;
};

constexpr int ERR_CONVERT = 41, ERR_MMA = 42, ERR_SOFTMAX = 43, ERR_LAYOUT = 44, ERR_LOADER = 45;

// EXTRAS: whether a window, blocks of positions, a sink or a gate may be asked for; without them their code is
// not there.  gridDim.z blocks (a cluster) share a tile's key blocks.
template <bool EXTRAS>
__global__ void __launch_bounds__(NUM_THREADS, 1) cache8_prompt_kernel(const __grid_constant__ CUtensorMap pool_map, const AttnArgs a) {
  const AttentionExtras extras = EXTRAS ? a.extras : AttentionExtras{0, nullptr, nullptr, 0};
  const int window = EXTRAS ? a.window : 0;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles need 1024-byte alignment (checked below)
  uint8_t* q_smem = smem;                              // [TILES][KA sub-tiles]
  uint8_t* ring = q_smem + TILES * Q_BYTES;            // [SLOTS][KA sub-tiles]: key and value tiles in turn
  uint8_t* raw_ring = ring + SLOTS * TILE_BYTES;       // [RAW_SLOTS]: the same tiles as codes
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + TILES_BYTES);
  uint64_t* tile_full = bars;               // [SLOTS] converters -> MMA (and softmax): the slot's tile is written
  uint64_t* tile_empty = tile_full + SLOTS; // [SLOTS] both MMA issuers (commit) -> converters
  uint64_t* raw_full = tile_empty + SLOTS;  // [RAW_SLOTS] loader -> converters: the slot's codes have landed
  uint64_t* raw_empty = raw_full + RAW_SLOTS; // [RAW_SLOTS] converters -> loader
  uint64_t* q_full = raw_empty + RAW_SLOTS; // [2] softmax group -> MMA: Q_g staged
  uint64_t* s_full = q_full + 2;            // [2][2] MMA (commit) -> softmax, per group and half of 64 keys
  uint64_t* p_full = s_full + 4;            // [2][2] softmax -> MMA: half h of P written
  uint64_t* pv_done = p_full + 4;           // [2][2] MMA (commit) -> softmax, MMA: the product with half h is complete
  uint64_t* known = pv_done + 4;            // [EXPONENTS] loader -> softmax: a key block's exponents
  int2* exponents = reinterpret_cast<int2*>(known + EXPONENTS);   // [EXPONENTS] of a key block's keys and values
  uint32_t* factors = reinterpret_cast<uint32_t*>(exponents + EXPONENTS);   // [RAW_SLOTS][BLOCKS] what is left of a scale, twice as a half; 0: zeros
  uint32_t* tmem_slot = factors + RAW_SLOTS * BLOCKS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // ---- what this block works on (uniform across the cluster).  The step's lists are there before its kernels start, so they may
  // be read ahead of pdl_wait().  Blocks are handed out with x fastest: all key/value heads of the latest tile first (it sees
  // the most keys), then of the tile before it, ...
  const int tile = gridDim.y - 1 - blockIdx.y, kvh = blockIdx.x;
  const int seq = a.lists.tile_seq[tile];
  if (seq < 0) {
    pdl_wait();
    return;
  }
  if (smem_u32(smem) & 1023) {   // never seen; refuse rather than compute with a broken layout
    if (threadIdx.x == 0) atomicCAS(a.error_word, 0, ERR_LAYOUT);
    return;
  }
  const int group = a.q_heads / a.cache.kv_heads;
  const int q_start = a.lists.seq_q_start[seq], q_len = a.lists.seq_q_len[seq], kv_len = a.lists.seq_kv_len[seq];
  const int row0 = a.lists.tile_index[tile] * BLOCK_ROWS, n_rows = q_len * group, pos0 = kv_len - q_len;
  // per group (tile of 128 rows): its key blocks [g_lo, g_hi) and the positions of its first and last row
  int g_lo[TILES] = {}, g_hi[TILES] = {}, g_min_pos[TILES] = {}, g_max_pos[TILES] = {};
  int kb_lo = 1 << 30, kb_hi = 0;   // the union of the two ranges, then this block's share of it
#pragma unroll
  for (int g = 0; g < TILES; ++g) {
    const int first_row = row0 + g * BM;
    if (first_row >= n_rows) continue;
    g_min_pos[g] = pos0 + first_row / group;
    g_max_pos[g] = pos0 + min(q_len - 1, (first_row + BM - 1) / group);
    g_lo[g] = first_visible_key(g_min_pos[g], window, extras.chunk) / BN;
    g_hi[g] = g_max_pos[g] / BN + 1;
    kb_lo = min(kb_lo, g_lo[g]);
    kb_hi = max(kb_hi, g_hi[g]);
  }
  const int n_splits = gridDim.z, split = blockIdx.z;
  if (n_splits > 1) {
    const int n = kb_hi - kb_lo, from = kb_lo + n * split / n_splits;
    kb_hi = kb_lo + n * (split + 1) / n_splits;
    kb_lo = from;
#pragma unroll
    for (int g = 0; g < TILES; ++g) {
      g_lo[g] = max(g_lo[g], kb_lo);
      g_hi[g] = max(g_lo[g], min(g_hi[g], kb_hi));
    }
  }
  const int n_kb = kb_hi - kb_lo;

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&pool_map)) : "memory");
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&tile_full[s], CONVERT_THREADS / 32);
      mbar_init(&tile_empty[s], TILES);
    }
    for (int s = 0; s < EXPONENTS; ++s) mbar_init(&known[s], 1);
    for (int s = 0; s < RAW_SLOTS; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], CONVERT_THREADS / 32);
    }
    for (int b = 0; b < 2; ++b) mbar_init(&q_full[b], GROUP_THREADS);
    for (int b = 0; b < 4; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], GROUP_THREADS);
      mbar_init(&pv_done[b], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();      // (the MMA issuer too: the limit of its waits counts from here)

  // What a softmax thread carries to the end: its row's state.
  const int g = (warp >> 2) & 1, r = (warp & 3) * 32 + lane, R = row0 + g * BM + r;     // warps 0-7
  const bool row_valid = R < n_rows;
  const int token = row_valid ? R / group : 0, head = row_valid ? kvh * group + R % group : 0;
  const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16), o_addr = lane_addr + O_COL + g * D;
  float m = -INFINITY, l = 0.0f;
  const int my_lo = g ? g_lo[1] : g_lo[0], my_n = (g ? g_hi[1] : g_hi[0]) - my_lo;

  if (warp >= CONVERT_WARP && warp < MMA_WARP) {
    // ------------------------------------------------------------------ converters
    // A thread takes 16 codes (a chunk) of CHUNKS rows.  The eight threads whose accesses share a turn of the banks hold four chunks of two rows
    // that meet eight different bank groups, in the codes as they lie and in the halves as they are written: neighbours at head size 64, rows
    // that differ in bits 0 and 2 at 128.
    const int cw = warp - CONVERT_WARP;
    const int chunk = D == 128 ? (cw >> 1) * 4 + (lane & 3) : lane & 3;
    const int row_in = D == 128 ? (cw & 1) * 8 + ((lane >> 3) ^ ((lane >> 2) & 1) * 5) : cw * 8 + (lane >> 2);
    constexpr int STEP = BN / CHUNKS;             // rows from one of a thread's chunks to the next: one or two scale blocks
    bool ok = true;
    for (int n = 0; n < 2 * n_kb; ++n) {
      const int raw_slot = n % RAW_SLOTS, slot = n % SLOTS, use = n / SLOTS;
      ok = mbar_wait(&raw_full[raw_slot], (uint32_t)(n / RAW_SLOTS) & 1u, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint4 raw[CHUNKS];
      uint32_t factor[CHUNKS];
      const uint32_t from = smem_u32(raw_ring) + raw_slot * RAW_BYTES;
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        const int row = row_in + i * STEP;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[i].x), "=r"(raw[i].y), "=r"(raw[i].z), "=r"(raw[i].w) : "r"(from + raw_swizzled(row, chunk)) : "memory");
        factor[i] = factors[raw_slot * BLOCKS + row / SCALE_TOKENS];      // the same for the whole warp
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&raw_empty[raw_slot]);
      ok = use == 0 || mbar_wait(&tile_empty[slot], (uint32_t)(use - 1) & 1u, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint32_t to = smem_u32(ring) + slot * TILE_BYTES + (chunk >> 2) * SUB;
      const int behind = kv_len - (kb_lo + (n >> 1)) * BN;       // rows from here on lie behind the request's last key
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        const int row = row_in + i * STEP;
        uint32_t w[8];
        halves(raw[i].x, w[0], w[1]);
        halves(raw[i].y, w[2], w[3]);
        halves(raw[i].z, w[4], w[5]);
        halves(raw[i].w, w[6], w[7]);
        if (factor[i] != 0x3c003c00u) {
          // (where no page is held, or a scale is lost beside a far larger one, zeros; whatever lay there may be NaN)
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = factor[i] ? mul_half2(w[k], factor[i]) : 0u;
        }
        if (row >= behind) {     // masked as keys, but as values zero times whatever lies there must be zero
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = 0u;
        }
        const int first = (chunk & 3) * 2;
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + swizzled(row, first)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + swizzled(row, first + 1)), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&tile_full[slot]);
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      atomicCAS(a.error_word, 0, ERR_CONVERT);
    }
  } else if (warp == LOADER_WARP) {
    // ------------------------------------------------------------------ loader
    // Lane b looks after the key block's scale block b.  Pages are looked up two key blocks ahead and scales one, so that neither is waited for.
    auto find_page = [&](int jj) {      // -1: not held, or wholly behind the request's last key
      const int key = (kb_lo + jj) * BN + lane * SCALE_TOKENS;
      return lane < BLOCKS && jj < n_kb && key < kv_len ? page_of(a.cache, seq, key) : -1;
    };
    struct Place {
      long long row;           // of the pool, without the cache's own offset, or -1
      float k_scale, v_scale;
    };
    auto place = [&](int jj, int page) {
      Place p{-1, 0.0f, 0.0f};
      if (page >= 0) {
        const int in_page = ((kb_lo + jj) * BN + lane * SCALE_TOKENS) % a.cache.page_tokens;
        p.row = (long long)page * a.page_rows + (long long)kvh * a.cache.page_tokens + in_page;
        const long long at = (long long)page * a.cache.scale_stride + (long long)kvh * (a.cache.page_tokens / SCALE_TOKENS) + in_page / SCALE_TOKENS;
        p.k_scale = __ldcg(a.cache.k_scale + at);
        p.v_scale = __ldcg(a.cache.v_scale + at);
      }
      return p;
    };
    // What is left of the lane's scale once the largest exponent of the key block is taken out, and that exponent.
    auto split_scale = [&](const Place& p, float scale, int& most) {
      const bool lost = isnan(scale), there = p.row >= 0 && !lost;
      const int e = there ? exponent_of(scale) : -1000;
      most = __reduce_max_sync(0xffffffffu, e);
      if (most == -1000) most = 0;
      return p.row < 0 ? 0u : lost ? 0x7e007e00u : half_power(most - e);
    };
    const int per_piece = a.box_rows / SCALE_TOKENS;
    const bool leads = lane < BLOCKS && lane % per_piece == 0;      // a piece of a page is its first scale block's lane's to copy
    bool ok = true;
    int issued = 0;
    Place now = place(0, find_page(0));
    int page = find_page(1);
    for (int jj = 0; jj < n_kb && ok; ++jj) {
      const Place next = place(jj + 1, page);
      page = find_page(jj + 2);
      int ek, ev;
      const uint32_t fk = split_scale(now, now.k_scale, ek), fv = split_scale(now, now.v_scale, ev);
      if (lane == 0) {
        exponents[jj % EXPONENTS] = make_int2(ek, ev);
        mbar_arrive(&known[jj % EXPONENTS]);
      }
      const uint32_t copies = __popc(__ballot_sync(0xffffffffu, leads && now.row >= 0));
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const int n = 2 * jj + which, slot = n % RAW_SLOTS, use = n / RAW_SLOTS;
        ok = ok && (use == 0 || mbar_wait(&raw_empty[slot], (uint32_t)(use - 1) & 1u, abort_flag));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane < BLOCKS) factors[slot * BLOCKS + lane] = which ? fv : fk;
        __syncwarp();
        if (lane == 0) mbar_expect_tx(&raw_full[slot], copies * a.box_rows * D);   // also the one arrival
        __syncwarp();
        if (leads && now.row >= 0)
          tma_load_2d(smem_u32(raw_ring) + slot * RAW_BYTES + lane * SCALE_TOKENS * D, &pool_map, &raw_full[slot], 0,
                      (int)(now.row + (which ? a.v_row0 : a.k_row0)));
        issued = n + 1;
      }
      now = next;
    }
    if (!ok) {
      if (lane == 0) {
        *abort_flag = 1;
        atomicCAS(a.error_word, 0, ERR_LOADER);
        // this block's copies in flight land before it leaves (the waits of the others end at the flag)
        volatile int never = 0;
        for (int n = max(0, issued - RAW_SLOTS); n < issued; ++n) mbar_wait(&raw_full[n % RAW_SLOTS], (uint32_t)(n / RAW_SLOTS) & 1u, &never);
      }
      __syncwarp();
    }
  } else if (warp < LOADER_WARP && warp >= MMA_WARP) {
    // ------------------------------------------------------------------ MMA issuers: one a tile, which waits for nothing that its tile does not
    // need (a single one that asked for both tiles' events in turn took about 1,000 cycles from an event to its product)
    if (n_kb > 0 && elect_one()) {
      constexpr uint32_t idesc_s = instr_desc(BM, S_PIECE, 0);
      constexpr uint32_t idesc_o = instr_desc(BM, D, 1);
      const int g = warp - MMA_WARP, lo = (g ? g_lo[1] : g_lo[0]) - kb_lo, hi = (g ? g_hi[1] : g_hi[0]) - kb_lo;   // of the block's key blocks, its
      const uint32_t s_tmem = tmem_base + g * BN, o_tmem = tmem_base + O_COL + g * D;
      const uint64_t q_desc = smem_desc_sw128(smem_u32(q_smem) + g * Q_BYTES);
      bool ok = true;
      auto landed = [&](int n) { return mbar_wait(&tile_full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u, abort_flag); };
      // half h of S_g = Q_g K(jj)^T
      auto issue_s = [&](int jj, int h) {
        const int slot = (2 * jj) % SLOTS, i = jj - lo;
        ok = ok && (h > 0 || landed(2 * jj)) && (i > 0 ? mbar_wait(&pv_done[g * 2 + h], (uint32_t)(i - 1) & 1u, abort_flag)   // P(i - 1) has been read
                                                       : h > 0 || mbar_wait(&q_full[g], 0, abort_flag));
        if (!ok) return;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t k_desc = smem_desc_sw128(smem_u32(ring) + slot * TILE_BYTES + h * S_PIECE * 128);
#pragma unroll
        for (int at = 0; at < KA; ++at)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_ss(s_tmem + h * S_PIECE, q_desc + (at * SUB >> 4) + 2 * k, k_desc + (at * SUB >> 4) + 2 * k, idesc_s, (at > 0 || k > 0) ? 1u : 0u);
        umma_commit(&s_full[g * 2 + h]);
        if (h == 1) umma_commit(&tile_empty[slot]);
      };
      // O_g (+)= half h of P_g V(jj): the group's O accumulates in tensor memory over its key blocks
      auto issue_pv = [&](int jj, int h) {
        const int slot = (2 * jj + 1) % SLOTS, i = jj - lo;
        ok = ok && (h > 0 || landed(2 * jj + 1)) && mbar_wait(&p_full[g * 2 + h], (uint32_t)i & 1u, abort_flag);
        if (!ok) return;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t v_desc = smem_desc_sw128(smem_u32(ring) + slot * TILE_BYTES, SUB);
#pragma unroll
        for (int kk = 0; kk < S_PIECE / 16; ++kk)
          umma_ts(o_tmem, s_tmem + h * S_PIECE + kk * 8, v_desc + (uint64_t)((h * (S_PIECE / 16) + kk) * 2048 >> 4), idesc_o,
                  (kk > 0 || h > 0 || i > 0) ? 1u : 0u);
        umma_commit(&pv_done[g * 2 + h]);
        if (h == 1) umma_commit(&tile_empty[slot]);
      };
      auto pass = [&](int jj) {       // a key block that only the other tile reads
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          ok = ok && landed(2 * jj + which);
          if (ok) mbar_arrive(&tile_empty[(2 * jj + which) % SLOTS]);
        }
      };
      for (int jj = 0; jj < (lo < hi ? lo : n_kb) && ok; ++jj) pass(jj);
      if (lo < hi) {
        issue_s(lo, 0);
        issue_s(lo, 1);
        for (int jj = lo; jj < hi && ok; ++jj)
          for (int h = 0; h < 2; ++h) {
            issue_pv(jj, h);
            if (jj + 1 < hi) issue_s(jj + 1, h);
          }
        for (int jj = hi; jj < n_kb && ok; ++jj) pass(jj);
      }
      if (!ok) {
        *abort_flag = 1;
        atomicCAS(a.error_word, 0, ERR_MMA);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax: group g owns tile g, one thread per row
    float factor;       // scale * log2(e), times the power of two that was taken out of the row's queries
    {
      uint4 raw[D / 8];
#pragma unroll
      for (int c = 0; c < D / 8; ++c) raw[c] = make_uint4(0, 0, 0, 0);
      if (row_valid) {
        const uint4* src = reinterpret_cast<const uint4*>(a.q + ((long long)(q_start + token) * a.q_heads + head) * D);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) raw[c] = __ldg(src + c);
      }
      const __nv_bfloat162* pairs = reinterpret_cast<const __nv_bfloat162*>(raw);
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 2; ++i) most = fmaxf(most, fmaxf(fabsf(__low2float(pairs[i])), fabsf(__high2float(pairs[i]))));
      const int e = most > 0.0f ? min(max(exponent_of(most) - 10, -100), 116) : 0;     // the largest entry to [2^10, 2^11)
      const float down = power_of_two(-e);
      factor = a.scale_log2 * power_of_two(e);
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_half(__low2float(pairs[4 * c + i]) * down, __high2float(pairs[4 * c + i]) * down);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(q_smem) + g * Q_BYTES + (c >> 3) * SUB + swizzled(r, c & 7)),
                     "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mbar_arrive(&q_full[g]);
    const int row_pos = row_valid ? pos0 + token : -1;
    const uint32_t s_addr = lane_addr + g * BN;
    const int row_lo = first_visible_key(row_pos, window, extras.chunk);
    const int tile_min_pos = g ? g_min_pos[1] : g_min_pos[0];
    const int tile_max_lo = first_visible_key(g ? g_max_pos[1] : g_max_pos[0], window, extras.chunk);   // from here on no row's bound hides a key
    // the product with half h of this group's block k is complete
    auto wait_pv = [&](int k, int h) { return mbar_wait(&pv_done[g * 2 + h], (uint32_t)k & 1u, abort_flag); };
    bool ok = true;
    for (int i = 0; i < my_n && ok; ++i) {
      const int jj = my_lo + i - kb_lo, key0 = (my_lo + i) * BN;
      ok = mbar_wait(&known[jj % EXPONENTS], (uint32_t)(jj / EXPONENTS) & 1u, abort_flag);
      const int2 e = exponents[jj % EXPONENTS];
      const float c = factor * power_of_two(e.x), ev = (float)e.y;
      const bool all_visible = key0 + BN - 1 <= tile_min_pos && (!EXTRAS || key0 >= tile_max_lo);
      uint64_t l2[2] = {0, 0};      // the block's part of the sum, four parts of it
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ok = ok && mbar_wait(&s_full[g * 2 + h], (uint32_t)i & 1u, abort_flag) && !*abort_flag;
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t v[S_PIECE];
#pragma unroll
        for (int k = 0; k < S_PIECE; k += 32) tmem_load32_nowait(s_addr + h * S_PIECE + k, v + k);
        tmem_wait_loads();
        if (!all_visible) {
#pragma unroll
          for (int k = 0; k < S_PIECE; ++k) {
            const int key = key0 + h * S_PIECE + k;
            const bool visible = key <= row_pos && (!EXTRAS || key >= row_lo);
            if (!visible) v[k] = 0xff800000u;   // -inf: probability 0
          }
        }
        float mx0 = __uint_as_float(v[0]), mx1 = __uint_as_float(v[1]), mx2 = __uint_as_float(v[2]), mx3 = __uint_as_float(v[3]);
#pragma unroll
        for (int k = 4; k < S_PIECE - 4; k += 8) {   // four independent partial maxima
          mx0 = max3(mx0, __uint_as_float(v[k]), __uint_as_float(v[k + 1]));
          mx1 = max3(mx1, __uint_as_float(v[k + 2]), __uint_as_float(v[k + 3]));
          mx2 = max3(mx2, __uint_as_float(v[k + 4]), __uint_as_float(v[k + 5]));
          mx3 = max3(mx3, __uint_as_float(v[k + 6]), __uint_as_float(v[k + 7]));
        }
        mx0 = max3(mx0, __uint_as_float(v[S_PIECE - 4]), __uint_as_float(v[S_PIECE - 3]));
        mx1 = max3(mx1, __uint_as_float(v[S_PIECE - 2]), __uint_as_float(v[S_PIECE - 1]));
        const float m_new = fmaxf(m, fmaf(fmaxf(max3(mx0, mx1, mx2), mx3), c, ev));   // c > 0: the maximum commutes with it
        // tensor-memory loads and stores are warp-wide: the warp moves its maxima together, as soon as one of
        // its rows has outgrown its own by the step (a row that has not may follow the true maximum just as well)
        const bool move = __any_sync(0xffffffffu, m_new > m + RESCALE_STEP);
        if (move) {
          const float corr = fast_exp2(m - (m_new == -INFINITY ? 0.0f : m_new));   // m = -inf gives 0
          m = m_new;
          l *= corr;
          l2[0] = fma2(l2[0], pair(corr, corr), 0);
          l2[1] = fma2(l2[1], pair(corr, corr), 0);
          if (i > 0 || h > 0) {     // O = O * corr in tensor memory, when every product issued so far is complete
            if (!(h > 0 ? wait_pv(i, 0) : wait_pv(i - 1, 1))) {
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
              uint32_t t[32];
              tmem_load32_nowait(o_addr + c0, t);
              tmem_wait_loads();
#pragma unroll
              for (int k = 0; k < 32; ++k) t[k] = __float_as_uint(__uint_as_float(t[k]) * corr);
              tmem_store32(o_addr + c0, t);
            }
          }
        }
        const float shift = ev - (m == -INFINITY ? 0.0f : m);
        const uint64_t c2 = pair(c, c), shift2 = pair(shift, shift);
        uint32_t packed[S_PIECE / 2];
#pragma unroll
        for (int k = 0; k < S_PIECE; k += 2) {
          float x0, x1;
          unpair(fma2(pair(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), c2, shift2), x0, x1);
          const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
          l2[k / 2 % 2] = add2(l2[k / 2 % 2], pair(p0, p1));
          packed[k / 2] = pack_half(p0, p1);
        }
        tmem_store32(s_addr + h * S_PIECE, packed);      // over the scores that it was made of
        tmem_wait_stores();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&p_full[g * 2 + h]);
      }
      if (!ok) break;
      float part0, part1;
      unpair(add2(l2[0], l2[1]), part0, part1);
      l = fmaf(part0 + part1, power_of_two(-e.y), l);
    }
    if (ok && my_n > 0) ok = wait_pv(my_n - 1, 1) && !*abort_flag;
    if (!ok) {
      *abort_flag = 1;
      atomicCAS(a.error_word, 0, ERR_SOFTMAX);
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (n_splits == 1 && ok && my_n > 0) {
      // ---- every thread finishes its own row: O / l out of tensor memory, rounded to bfloat16, 64 bytes
      // at a time.  Heads that share a key/value head lie side by side in a token's output row, as their
      // rows do in the tile.  (The loads are warp-wide, so rows without an output still take part.)
      // the sink joins the sum, taken against the same maximum (far above it the sum is infinite, the row zero)
      if (extras.sink && row_valid) l += exp2f(sink_log2(extras, head) - m);
      const float inv = l == 0.0f ? 0.0f : (row_valid ? head_gate<__nv_bfloat16>(extras, q_start + token, head) : 1.0f) / l;
      uint4* dst = reinterpret_cast<uint4*>(a.out + ((long long)(q_start + token) * a.q_heads + head) * D);
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t t[32];
        tmem_load32_nowait(o_addr + c0, t);
        tmem_wait_loads();
        if (row_valid) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            dst[c0 / 8 + k] = make_uint4(pack_bf16(__uint_as_float(t[8 * k]) * inv, __uint_as_float(t[8 * k + 1]) * inv),
                                         pack_bf16(__uint_as_float(t[8 * k + 2]) * inv, __uint_as_float(t[8 * k + 3]) * inv),
                                         pack_bf16(__uint_as_float(t[8 * k + 4]) * inv, __uint_as_float(t[8 * k + 5]) * inv),
                                         pack_bf16(__uint_as_float(t[8 * k + 6]) * inv, __uint_as_float(t[8 * k + 7]) * inv));
        }
      }
    }
  }
  if (n_splits > 1) {
    // ---- every row's state into this block's shared memory (over the tiles, which no product reads any more), then the rows
    // r % n_splits == split merged over the cluster's blocks in index order
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    float* states = reinterpret_cast<float*>(smem);        // [BLOCK_ROWS][STATE]
    if (warp < CONVERT_WARP) {
      float* row = states + (size_t)(g * BM + r) * STATE;
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t t[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) t[k] = 0u;
        if (my_n > 0) {      // the same for the whole group
          tmem_load32_nowait(o_addr + c0, t);
          tmem_wait_loads();
        }
#pragma unroll
        for (int k = 0; k < 32; k += 4)
          *reinterpret_cast<float4*>(row + c0 + k) = make_float4(__uint_as_float(t[k]), __uint_as_float(t[k + 1]), __uint_as_float(t[k + 2]),
                                                                 __uint_as_float(t[k + 3]));
      }
      *reinterpret_cast<float4*>(row + D) = make_float4(m, l, 0.0f, 0.0f);
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int i = threadIdx.x; i < BLOCK_ROWS / n_splits * (D / 4); i += NUM_THREADS) {
      const int row = i / (D / 4) * n_splits + split, c4 = i % (D / 4), packed = row0 + row;
      if (packed >= n_rows) continue;
      const int tok = packed / group, hd = kvh * group + packed % group;
      const uint32_t local = smem_u32(states + (size_t)row * STATE);
      const float sink = sink_log2(extras, hd);
      float M = sink;
      for (int z = 0; z < n_splits; ++z) M = fmaxf(M, load_peer4(peer_smem(local, z) + D * 4).x);
      const float M_use = M == -INFINITY ? 0.0f : M;
      float L = exp2f(sink - M_use);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int z = 0; z < n_splits; ++z) {
        const uint32_t from = peer_smem(local, z);
        const float4 ml = load_peer4(from + D * 4), v = load_peer4(from + c4 * 16);
        const float f = ml.x == -INFINITY ? 1.0f : exp2f(ml.x - M_use);      // without a maximum: zeros, or NaN to be handed on
        L += ml.y * f;
        acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
      }
      const float inv = L == 0.0f ? 0.0f : head_gate<__nv_bfloat16>(extras, q_start + tok, hd) / L;
      *reinterpret_cast<uint2*>(a.out + ((long long)(q_start + tok) * a.q_heads + hd) * D + c4 * 4) =
          make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // others may still read this block's states
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

}  // namespace

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}

extern "C" int llm_cache8_attention_prompt_rows() { return BLOCK_ROWS; }

// Writes the 128-byte tensor map of a pool of `rows` rows of D codes starting at `base` (16-byte aligned), boxes of `box_rows` whole rows
// (the largest power of two that divides the page size, up to 128), swizzled as raw_swizzled says.
extern "C" int llm_cache8_prompt_pool_map(void* map_out, const void* base, long long rows, int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return 1000 + (int)cudaErrorNotSupported;
  if ((reinterpret_cast<uintptr_t>(base) & 15) || rows <= 0 || rows > 0x7fffffffLL || box_rows < SCALE_TOKENS || BN % box_rows) return ERR_BAD_SIZE;
  cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)D};
  cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)box_rows};
  cuuint32_t elem[2] = {1, 1};
  CUresult r = fn(reinterpret_cast<CUtensorMap*>(map_out), CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 2000 + (int)r;
}

// The tiles of llm_step_maps with tile_rows = llm_cache8_attention_prompt_rows() (entries of -1 return at once); n_splits (1, 2, 4 or 8)
// blocks share a tile's keys.  `pool_map`: llm_cache8_prompt_pool_map over `pool_base`, in which the cache's codes lie, with boxes of
// `box_rows` rows, which divide the page size.  chunk, sink, gate and gate_stride (elements): `AttentionExtras`; 0 and null: none.
extern "C" int llm_cache8_attention_prompt(const void* q, void* out, const Cache8* cache, const void* pool_map, const void* pool_base,
                                           int box_rows, const StepLists* lists, int n_splits, int q_heads,
                                           float scale, int window, int chunk, const float* sink, const void* gate,
                                           long long gate_stride, int* error_word, cudaStream_t stream) {
  const int n_tiles = lists->n_tiles;
  if (n_tiles <= 0) return 0;
  const Cache8& c = *cache;
  if (c.head_dim != D || c.kv_heads <= 0 || q_heads <= 0 || q_heads % c.kv_heads || c.page_tokens <= 0 || c.page_tokens % SCALE_TOKENS ||
      n_tiles > 65535 || !(scale > 0.0f) || (n_splits != 1 && n_splits != 2 && n_splits != 4 && n_splits != 8))
    return ERR_BAD_SIZE;
  const uintptr_t all = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(c.k) |
                        reinterpret_cast<uintptr_t>(c.v) | (uintptr_t)c.page_stride;
  const long long k_off = reinterpret_cast<const char*>(c.k) - reinterpret_cast<const char*>(pool_base);
  const long long v_off = reinterpret_cast<const char*>(c.v) - reinterpret_cast<const char*>(pool_base);
  if ((all & 15) || k_off < 0 || v_off < 0 || k_off % D || v_off % D || c.page_stride % D) return ERR_BAD_ALIGN;
  if (box_rows < SCALE_TOKENS || BN % box_rows || box_rows % SCALE_TOKENS || c.page_tokens % box_rows) return ERR_BAD_SIZE;
  static bool configured = false;
  if (!configured) {
    if (cudaFuncSetAttribute(cache8_prompt_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(cache8_prompt_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES) != cudaSuccess)
      return launch_status();
    configured = true;
  }
  const AttnArgs a{reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<__nv_bfloat16*>(out), c, c.page_stride / D, k_off / D, v_off / D,
                   box_rows, *lists, q_heads,
                   scale * 1.4426950408889634f, window, AttentionExtras{chunk, sink, gate, gate_stride}, error_word};
  CUtensorMap map;   // the caller's buffer need not be 64-byte aligned
  memcpy(&map, pool_map, sizeof(CUtensorMap));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c.kv_heads, n_tiles, n_splits);
  cfg.blockDim = dim3(NUM_THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n_attr = 0;
  if (n_splits > 1) {
    attr[n_attr].id = cudaLaunchAttributeClusterDimension;
    attr[n_attr].val.clusterDim.x = 1;
    attr[n_attr].val.clusterDim.y = 1;
    attr[n_attr].val.clusterDim.z = n_splits;
    ++n_attr;
  }
  if (pdl_enabled()) {
    attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
    ++n_attr;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n_attr;
  cudaLaunchKernelEx(&cfg, window > 0 || chunk > 0 || sink || gate ? cache8_prompt_kernel<true> : cache8_prompt_kernel<false>, map, a);
  return launch_status();
}
