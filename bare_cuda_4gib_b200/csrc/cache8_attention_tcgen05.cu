// Softmax attention of prompt portions over a cache of e4m3 codes (cache8.cuh) on the Blackwell tensor cores: what
// attention_tcgen05.cu is to a bfloat16 cache, for requests with more than 16 packed rows (tokens x query heads of one key/value
// head).  Nothing of cuongvng/bare-cuda-4gib's [heads, T, keys] score buffer exists (engine/kernels/attention_qk.cu:49-68,
// softmax.cu:28-42, attention_av.cu:24-44).
//
// One thread block = two tiles of 128 packed rows of one request and one key/value head, which share every key and value
// block.  Keys are visited in blocks of 128 positions:
//   converter warps  (four) fetch a tile's codes from the request's pages, 16 bytes a load and one tile ahead, and write
//                  code * scale as bfloat16 into 128-byte-swizzled shared memory.  A scale is a power of two, so that number is a
//                  bfloat16 exactly, and everything behind it is the bfloat16 kernel.  Key tiles and value tiles go through
//                  ONE ring of slots in the order K(0) V(0) K(1) V(1) ..., each slot given back by the commit of the last product that
//                  reads it;
//   MMA thread     S_g = Q_g K^T (M 128, N 128, K head size) into tile g's S columns of tensor memory;
//   softmax warps  a group of four warps per tile; group g owns tile g and sees every key block of it.
//                  First it stages Q_g with cp.async.  Then, one thread per row: read the row of S from tensor memory once, 64 columns
//                  at a time, scale, mask, running maximum and sum in float32 (base 2), write P as bfloat16 into swizzled
//                  shared memory (the A operand of the second product);
//   MMA thread     O_g (+)= P_g V (M 128, N 64 per 64 value columns, K 128): O accumulates in tensor memory over all key blocks;
//   softmax warps  the maximum that the exponentials are taken against follows the row's true maximum only when that
//                  has grown by more than 2^8; at the end every thread divides its row of O by its sum and stores it.
// A NaN scale (a block that was given a NaN) makes keys NaN, hence the scores of the rows that see them; hidden scores are replaced, not
// multiplied, and values are finite always.  Values behind the request's last key are written as zeros.
// Every mbarrier wait is bounded: on a timeout the thread sets the error word, all roles leave their loops, tensor memory is
// released and the block returns.
// One B200: a prompt of 2,048 tokens (32 / 4 heads of 64) 50.0 us, 2,048 tokens behind 2,048 (32 heads of 128) 231.7 us.

#include "cache8.cuh"

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
constexpr int SUB = 128 * 128;   // bytes of a [128 rows x 64 bf16] swizzled sub-tile
constexpr int Q_BYTES = KA * SUB;        // one tile's queries
constexpr int TILE_BYTES = KA * SUB;     // one key tile or one value tile
constexpr int P_BYTES = 2 * SUB;         // [128 rows x 128 keys] as two sub-tiles
constexpr int SLOTS = HEAD_DIM == 64 ? 6 : 3;   // key and value tiles in flight (what shared memory allows)
constexpr int SOFTMAX_THREADS = 128 * TILES, CONVERT_THREADS = 128;
constexpr int MMA_WARP = SOFTMAX_THREADS / 32;
constexpr int NUM_THREADS = SOFTMAX_THREADS + 32 + CONVERT_THREADS;   // warps 0-7 softmax, 8 MMA, 9-12 converters
constexpr int TMEM_COLS = 256 * TILES;
constexpr int O_COL = TILES * BN;  // first tensor-memory column of the P V results (the S buffers lie before it)
constexpr int GROUP_THREADS = 128;
constexpr int S_PIECE = 64;      // columns of S a softmax thread holds in registers at a time (one sub-tile of P)
constexpr unsigned long long WAIT_LIMIT_NS = 1000000000ull;
constexpr size_t SMEM_BYTES = TILES * Q_BYTES + SLOTS * TILE_BYTES + TILES * P_BYTES + 256;   // 2 * SLOTS + 10 barriers, 2 words
// What a converter thread fetches of a tile: 16 codes (chunk ct % CHUNKS) of rows ct / CHUNKS + i * STRIDE, i < CHUNKS.
constexpr int CHUNKS = D / 16, STRIDE = CONVERT_THREADS / CHUNKS;
constexpr int BLOCKS = BN / SCALE_TOKENS;   // scale blocks of a key block

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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int bytes = valid ? 16 : 0;  // 0: the 16 bytes are filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Byte offset of the 16-byte chunk `chunk` (0..7) of row `row` inside a [rows x 64 bf16] sub-tile
// with the 128-byte swizzle: rows are 128 bytes, groups of 8 rows are 1024 bytes, and the chunk
// index is XORed with the row's index inside its group.
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
  return (uint32_t)((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4));
}

// Shared-memory matrix descriptor, 128-byte swizzle, 1024 bytes between 8-row groups.
__device__ __forceinline__ uint64_t smem_desc_sw128(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// float32 accumulator, bfloat16 operands, A K-major; B K-major or (b_mn = 1) MN-major.
__host__ __device__ constexpr uint32_t instr_desc(int m, int n, int b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_bf16(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
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
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}


struct AttnArgs {
  const __nv_bfloat16* q;      // [tokens, q_heads, D]
  __nv_bfloat16* out;          // [tokens, q_heads * D]
  Cache8 cache;
  const int32_t* seq_q_start;
  const int32_t* seq_q_len;
  const int32_t* seq_kv_len;
  const int32_t* tile_seq;     // per tile: batch sequence (-1: nothing to do)
  const int32_t* tile_index;   // per tile: which tile of BLOCK_ROWS of the sequence's packed rows
  int q_heads;
  float scale_log2;
  int window;
  AttentionExtras extras;
  int* error_word;
};

// Four codes as bfloat16 numbers: a code's exponent and fraction four places to the right are a bfloat16 2^120 times too small
// (its subnormals included), which the factor f1 = 2^(120 + e) mends; f2 (1 but for scales above 2^7) is the rest of the scale.
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ void bf16_of_codes(uint32_t codes, uint32_t f1, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = __byte_perm(codes, 0, 0x1404), b = __byte_perm(codes, 0, 0x3424);
  lo = mul_bf16x2((a & 0x80008000u) | ((a >> 4) & 0x07f007f0u), f1);
  hi = mul_bf16x2((b & 0x80008000u) | ((b >> 4) & 0x07f007f0u), f1);
}

constexpr int ERR_CONVERT = 41, ERR_MMA = 42, ERR_SOFTMAX = 43, ERR_LAYOUT = 44;

// EXTRAS: whether a window, blocks of positions, a sink or a gate may be asked for; without them their code is
// not there.
template <bool EXTRAS>
__global__ void __launch_bounds__(NUM_THREADS, 1) cache8_prompt_kernel(const AttnArgs a) {
  const AttentionExtras extras = EXTRAS ? a.extras : AttentionExtras{0, nullptr, nullptr, 0};
  const int window = EXTRAS ? a.window : 0;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles need 1024-byte alignment (checked below)
  uint8_t* q_smem = smem;                              // [TILES][KA sub-tiles]
  uint8_t* ring = q_smem + TILES * Q_BYTES;            // [SLOTS][KA sub-tiles]: key and value tiles in turn
  uint8_t* p_smem = ring + SLOTS * TILE_BYTES;         // [TILES][two sub-tiles of 64 keys]
  uint64_t* bars = reinterpret_cast<uint64_t*>(p_smem + TILES * P_BYTES);
  uint64_t* tile_full = bars;               // [SLOTS] converters -> MMA: the slot's tile is written
  uint64_t* tile_empty = tile_full + SLOTS; // [SLOTS] MMA (commit) -> converters
  uint64_t* q_full = tile_empty + SLOTS;    // [2] softmax group -> MMA: Q_g staged
  uint64_t* s_full = q_full + 2;            // [2] MMA (commit) -> softmax, per group
  uint64_t* p_full = s_full + 2;            // [2] softmax -> MMA: P written, per group
  uint64_t* o_full = p_full + 2;            // [2] MMA (commit) -> softmax, per group: P(i) V is complete
  uint64_t* s_free = o_full + 2;            // [2] softmax -> MMA: the group holds its S values in registers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_free + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023) {   // never seen; refuse rather than compute with a broken layout
    if (threadIdx.x == 0) atomicCAS(a.error_word, 0, ERR_LAYOUT);
    return;
  }
  // ---- what this block works on (uniform across the block).  The tile list and the requests'
  // lengths are written by the host before the step's first kernel, so they may be read ahead of
  // pdl_wait(); their latency then hides behind the barrier set-up and the tensor-memory allocation.
  // blocks are handed out with x fastest: all key/value heads of the latest tile first (it sees
  // the most keys), then of the tile before it, ... so the longest blocks of the whole grid start first
  const int tile = gridDim.y - 1 - blockIdx.y, kvh = blockIdx.x;
  const int seq = a.tile_seq[tile];
  int q_start = 0, q_len = 0, kv_len = 0, row0 = 0, n_rows = 0, pos0 = 0, group = 1;
  // per group (tile of 128 rows): its key blocks [g_lo, g_hi) and the positions of its first and last row
  int g_lo[TILES] = {}, g_hi[TILES] = {}, g_min_pos[TILES] = {}, g_max_pos[TILES] = {};
  int kb_lo = 0, n_kb = 0;   // the union of the two ranges: what the converters bring
  if (seq >= 0) {
    group = a.q_heads / a.cache.kv_heads;
    q_start = a.seq_q_start[seq];
    q_len = a.seq_q_len[seq];
    kv_len = a.seq_kv_len[seq];
    row0 = a.tile_index[tile] * BLOCK_ROWS;
    n_rows = q_len * group;
    pos0 = kv_len - q_len;
    int lo_all = 1 << 30, hi_all = 0;
#pragma unroll
    for (int g = 0; g < TILES; ++g) {
      const int first_row = row0 + g * BM;
      if (first_row >= n_rows) continue;
      const int first_token = first_row / group, last_token = min(q_len - 1, (first_row + BM - 1) / group);
      g_min_pos[g] = pos0 + first_token;
      g_max_pos[g] = pos0 + last_token;
      const int lo_key = first_visible_key(g_min_pos[g], window, extras.chunk);
      g_lo[g] = lo_key / BN;
      g_hi[g] = g_max_pos[g] / BN + 1;
      lo_all = min(lo_all, g_lo[g]);
      hi_all = max(hi_all, g_hi[g]);
    }
    if (hi_all > 0) kb_lo = lo_all, n_kb = hi_all - lo_all;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&tile_full[s], CONVERT_THREADS / 32);
      mbar_init(&tile_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&q_full[b], GROUP_THREADS);
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], GROUP_THREADS);
      mbar_init(&o_full[b], 1);
      mbar_init(&s_free[b], GROUP_THREADS);
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
  if (warp > MMA_WARP) {
    // ------------------------------------------------------------------ converters
    // Tile n of the ring is the keys (n even) or the values (n odd) of key block n / 2.  A tile's codes are asked for one tile ahead of
    // their conversion, and where a key block's scale blocks lie one tile before that.  Positions of no page (given back by a
    // window) and behind the request's last key become zeros: their keys are masked, but zero times whatever lies there must be zero.
    const int ct = threadIdx.x - (MMA_WARP + 1) * 32, chunk = ct % CHUNKS, row0 = ct / CHUNKS;
    struct Place {             // of a key block, lane b: its scale block b (the same for keys and values)
      long long at;            // codes from the cache's first, or -1
      float k_scale, v_scale;
    };
    auto look_up = [&](int jj) {
      Place p{-1, 0.0f, 0.0f};
      const int key = (kb_lo + jj) * BN + lane * SCALE_TOKENS;
      if (lane < BLOCKS && jj < n_kb && key < kv_len) {
        const int page = page_of(a.cache, seq, key);
        if (page >= 0) {
          const int in_page = key % a.cache.page_tokens;
          p.at = (long long)page * a.cache.page_stride + ((long long)kvh * a.cache.page_tokens + in_page) * D;
          const long long s = (long long)page * a.cache.scale_stride + (long long)kvh * (a.cache.page_tokens / SCALE_TOKENS) + in_page / SCALE_TOKENS;
          p.k_scale = __ldcg(a.cache.k_scale + s);
          p.v_scale = __ldcg(a.cache.v_scale + s);
        }
      }
      return p;
    };
    auto block_of = [&](int i) { return (row0 + i * STRIDE) / SCALE_TOKENS; };      // the same for a whole warp
    auto fetch = [&](uint4 (&raw)[CHUNKS], const Place& p, int n) {
      const uint8_t* base = (n & 1) ? a.cache.v : a.cache.k;
      const int key0 = (kb_lo + (n >> 1)) * BN;
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        const int row = row0 + i * STRIDE;
        const long long at = __shfl_sync(0xffffffffu, p.at, block_of(i));
        raw[i] = make_uint4(0, 0, 0, 0);
        if (at >= 0 && key0 + row < kv_len) raw[i] = __ldcg(reinterpret_cast<const uint4*>(base + at + (row % SCALE_TOKENS) * D + chunk * 16));
      }
    };
    auto convert = [&](const uint4 (&raw)[CHUNKS], const Place& p, int n) {
      const uint32_t base = smem_u32(ring) + (n % SLOTS) * TILE_BYTES + (chunk >> 2) * SUB;
      const float scale = (n & 1) ? p.v_scale : p.k_scale;
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        const int row = row0 + i * STRIDE;
        const float s = __shfl_sync(0xffffffffu, scale, block_of(i));
        const int e = exponent_of(s);
        const float f = isnan(s) ? s : power_of_two(min(max(e, SCALE_LEAST), 7) + 120);
        const uint32_t f1 = __byte_perm(__float_as_uint(f), 0, 0x3232);
        uint32_t w[8];
        bf16_of_codes(raw[i].x, f1, w[0], w[1]);
        bf16_of_codes(raw[i].y, f1, w[2], w[3]);
        bf16_of_codes(raw[i].z, f1, w[4], w[5]);
        bf16_of_codes(raw[i].w, f1, w[6], w[7]);
        if (e > 7) {           // rare, and the same for the whole warp
          const uint32_t f2 = __byte_perm(__float_as_uint(power_of_two(min(e, 127) - 7)), 0, 0x3232);
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = mul_bf16x2(w[k], f2);
        }
        // two 16-byte chunks of the row; threads of odd sub-tiles store theirs the other way round, so that the eight that share a row
        // (or two rows, at head size 64) meet eight different groups of banks
        const int first = (chunk & 3) * 2, swap = (chunk >> 2) & 1;
        const uint32_t at0 = base + swizzled(row, first + swap), at1 = base + swizzled(row, first + 1 - swap);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at0), "r"(swap ? w[4] : w[0]), "r"(swap ? w[5] : w[1]), "r"(swap ? w[6] : w[2]), "r"(swap ? w[7] : w[3]) : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at1), "r"(swap ? w[0] : w[4]), "r"(swap ? w[1] : w[5]), "r"(swap ? w[2] : w[6]), "r"(swap ? w[3] : w[7]) : "memory");
      }
    };
    bool ok = true;
    auto deliver = [&](const uint4 (&raw)[CHUNKS], const Place& p, int n) {
      const uint32_t use = (uint32_t)(n / SLOTS);   // how often the slot was filled before
      ok = ok && (use == 0 || mbar_wait(&tile_empty[n % SLOTS], (use - 1) & 1, abort_flag));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      convert(raw, p, n);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&tile_full[n % SLOTS]);
    };
    uint4 keys[CHUNKS], values[CHUNKS];
    Place now = look_up(0);
    if (n_kb > 0) fetch(keys, now, 0);
    for (int jj = 0; jj < n_kb && ok; ++jj) {
      fetch(values, now, 2 * jj + 1);
      const Place next = look_up(jj + 1);
      deliver(keys, now, 2 * jj);
      if (jj + 1 < n_kb) fetch(keys, next, 2 * jj + 2);
      deliver(values, now, 2 * jj + 1);
      now = next;
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      atomicCAS(a.error_word, 0, ERR_CONVERT);
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------------------------ MMA issuer
    if (n_kb > 0 && elect_one()) {
      constexpr uint32_t idesc_s = instr_desc(BM, BN, 0);
      constexpr uint32_t idesc_o = instr_desc(BM, 64, 1);
      auto active = [&](int g, int jj) { return kb_lo + jj >= g_lo[g] && kb_lo + jj < g_hi[g]; };
      // S_g = Q_g K(jj)^T into group g's S buffer; `last`: no product after this one reads the key tile
      auto issue_s = [&](int g, int jj, bool last) {
        const int slot = (2 * jj) % SLOTS;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t k_addr = smem_u32(ring) + slot * TILE_BYTES, q_addr = smem_u32(q_smem) + g * Q_BYTES;
#pragma unroll
        for (int at = 0; at < KA; ++at)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16(tmem_base + g * BN, smem_desc_sw128(q_addr + at * SUB) + 2 * k,
                      smem_desc_sw128(k_addr + at * SUB) + 2 * k, idesc_s, (at > 0 || k > 0) ? 1u : 0u);
        umma_commit(&s_full[g]);
        if (last) umma_commit(&tile_empty[slot]);
      };
      // O_g (+)= P_g V(jj): the group's O accumulates in tensor memory over its key blocks (`first`: overwrite)
      auto issue_pv = [&](int g, int jj, bool last, int i) {     // i: the group's i-th key block
        const int slot = (2 * jj + 1) % SLOTS;
        const bool first = i == 0;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t v_addr = smem_u32(ring) + slot * TILE_BYTES;
        const uint32_t p_addr = smem_u32(p_smem) + g * P_BYTES;
#pragma unroll
        for (int vt = 0; vt < KA; ++vt)
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            umma_bf16(tmem_base + O_COL + g * D + vt * 64, smem_desc_sw128(p_addr + (kk >> 2) * SUB) + 2 * (kk & 3),
                      smem_desc_sw128(v_addr + vt * SUB) + (uint64_t)(kk * 2048 >> 4), idesc_o, (kk > 0 || !first) ? 1u : 0u);
        umma_commit(&o_full[g]);
        if (last) umma_commit(&tile_empty[slot]);
      };
      // The two groups are served as they come: a group's next S as soon as it reports that it holds the
      // S before it in registers (and the key tile has landed), its P V as soon as it reports P (and has
      // read the O_block before).  Nothing is waited for while the other group could be served.
      bool ok = true;
      int s_next[TILES] = {}, pv_next[TILES] = {};      // per group: its next block to issue S / P V for
      int n_g[TILES];
#pragma unroll
      for (int g = 0; g < TILES; ++g) n_g[g] = g_hi[g] - g_lo[g];
      auto unfinished = [&]() {
        bool any = false;
#pragma unroll
        for (int g = 0; g < TILES; ++g) any = any || pv_next[g] < n_g[g];
        return any;
      };
      // Whether tile n has landed.  A barrier's parity tells one filling of a slot only from the one before it.
      // Groups that start with the same key block ask for the tiles as the slots are filled.  A group whose
      // first key block lies behind the other's (a window, or a later block of positions) would take an
      // earlier filling for its own: there the tiles are counted off in order.
      const bool counted = EXTRAS && g_lo[0] != g_lo[TILES - 1];
      int arrived = 0, arrived_slot = 0;
      uint32_t arrived_parity = 0;
      auto landed = [&](int n) {
        if (counted) {
          while (arrived <= n) {
            if (!mbar_try_wait(&tile_full[arrived_slot], arrived_parity)) return false;
            ++arrived;
            if (++arrived_slot == SLOTS) arrived_slot = 0, arrived_parity ^= 1u;
          }
          return true;
        }
        return mbar_try_wait(&tile_full[n % SLOTS], (n / SLOTS) & 1);
      };
      unsigned long long idle_since = 0;
      unsigned idle_spins = 0;
      while (ok && unfinished()) {
        bool progress = false;
#pragma unroll
        for (int g = 0; g < TILES; ++g) {
          const int o = 1 - g;   // the other group
          if (s_next[g] < n_g[g]) {
            const int i = s_next[g], jj = g_lo[g] + i - kb_lo;
            if ((i == 0 ? mbar_try_wait(&q_full[g], 0) : mbar_try_wait(&s_free[g], (i - 1) & 1)) && landed(2 * jj)) {
              // the other group is done with K(jj) if it never reads it or has issued its S for it already
              const bool last = !active(o, jj) || s_next[o] > kb_lo + jj - g_lo[o];
              issue_s(g, jj, last);
              s_next[g] = i + 1;
              progress = true;
            }
          }
          if (pv_next[g] < s_next[g]) {
            const int i = pv_next[g], jj = g_lo[g] + i - kb_lo;
            if (mbar_try_wait(&p_full[g], (uint32_t)i & 1u) && landed(2 * jj + 1)) {
              const bool last = !active(o, jj) || pv_next[o] > kb_lo + jj - g_lo[o];
              issue_pv(g, jj, last, i);
              pv_next[g] = i + 1;
              progress = true;
            }
          }
        }
        if (progress) {
          idle_spins = 0;
        } else if ((++idle_spins & 63u) == 0u) {
          if (idle_spins == 64u) idle_since = global_timer();
          if (*abort_flag || global_timer() - idle_since > WAIT_LIMIT_NS) ok = false;
        }
      }
      if (!ok) {
        *abort_flag = 1;
        atomicCAS(a.error_word, 0, ERR_MMA);
        for (int b = 0; b < TILES; ++b) umma_commit(&s_full[b]);   // release whoever waits
        for (int b = 0; b < TILES; ++b) umma_commit(&o_full[b]);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax: group g owns tile g, one thread per row
    const int quad = warp & 3, g = warp >> 2;        // tensor-memory lanes 32 * quad ..
    const int gt = threadIdx.x & (GROUP_THREADS - 1);
    const int tile_row0 = row0 + g * BM;
    // Q_g: 128 rows x D in 16-byte chunks, staged by the group's threads (a few chunks each, so one
    // round of global latency); rows past the request's packed rows are zero
    for (int i = gt; i < BM * (D / 8); i += GROUP_THREADS) {
      const int qr = i / (D / 8), c = i % (D / 8);
      const int QR = tile_row0 + qr;
      const bool valid = seq >= 0 && QR < n_rows;
      const int token = valid ? QR / group : 0, head = valid ? kvh * group + QR % group : 0;
      const __nv_bfloat16* src = a.q + ((long long)(q_start + token) * a.q_heads + head) * D + c * 8;
      cp_async16(smem_u32(q_smem) + g * Q_BYTES + (c >> 3) * SUB + swizzled(qr, c & 7), src, valid);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mbar_arrive(&q_full[g]);
    const int r = quad * 32 + lane;                  // row of the tile = tensor-memory lane
    const int R = tile_row0 + r;
    const bool row_valid = seq >= 0 && R < n_rows;
    const int row_pos = row_valid ? pos0 + R / group : -1;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_addr = lane_addr + g * BN, o_addr = lane_addr + O_COL + g * D;
    const int my_lo = g_lo[g], my_n = g_hi[g] - g_lo[g];
    const int row_lo = first_visible_key(row_pos, window, extras.chunk);
    const int tile_min_pos = g_min_pos[g];
    const int tile_max_lo = first_visible_key(g_max_pos[g], window, extras.chunk);   // from here on no row's bound hides a key
    // Running softmax of the row.  `m` is the maximum the exponentials are taken against; it follows the
    // true maximum only when that has grown by more than RESCALE_STEP (in base-2 units), so that O, which
    // accumulates in tensor memory over all key blocks, has to be rescaled rarely: with a stale maximum
    // the probabilities reach at most 2^RESCALE_STEP, and since sum and O are taken against the same `m`
    // their quotient is exact either way.
    constexpr float RESCALE_STEP = 8.0f;
    float m = -INFINITY, l = 0.0f;
    // this row of the group's P tiles (swizzled: chunk c of row r lies at c ^ (r % 8) inside the row's 128 bytes)
    const uint32_t p_row = smem_u32(p_smem) + g * P_BYTES + (r >> 3) * 1024 + (r & 7) * 128, p_xor = (uint32_t)(r & 7) << 4;
    // P(k) V of this group is complete
    auto wait_pv = [&](int k) { return mbar_wait(&o_full[g], (uint32_t)k & 1u, abort_flag); };
    bool ok = true;
    for (int i = 0; i < my_n && ok; ++i) {
      const int key0 = (my_lo + i) * BN;
      ok = mbar_wait(&s_full[g], i & 1, abort_flag) && !*abort_flag;
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const bool all_visible = key0 + BN - 1 <= tile_min_pos && (!EXTRAS || key0 >= tile_max_lo);
      // The row of S is read once, in two pieces of 64 columns (one sub-tile of P each).  Each piece
      // settles the maximum for itself: should the second piece move it, the probabilities of the
      // first, which this thread has just written, are rescaled where they lie (rare, as is every move).
      float l0 = 0.0f, l1 = 0.0f, l2 = 0.0f, l3 = 0.0f;
#pragma unroll
      for (int h = 0; h < BN / S_PIECE; ++h) {
        uint32_t v[S_PIECE];
#pragma unroll
        for (int c = 0; c < S_PIECE; c += 32) tmem_load32_nowait(s_addr + h * S_PIECE + c, v + c);
        tmem_wait_loads();
        if (h == BN / S_PIECE - 1) {   // the last read of S(i): the MMA thread may overwrite the buffer with S(i + 1)
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          mbar_arrive(&s_free[g]);
        }
        if (!all_visible) {
#pragma unroll
          for (int k = 0; k < S_PIECE; ++k) {
            const int key = key0 + h * S_PIECE + k;
            const bool visible = key <= row_pos && (!EXTRAS || key >= row_lo);
            if (!visible) v[k] = 0xff800000u;   // -inf: probability 0
          }
        }
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
        for (int k = 0; k < S_PIECE; k += 8) {   // four independent partial maxima
          mx0 = fmaxf(mx0, fmaxf(__uint_as_float(v[k]), __uint_as_float(v[k + 1])));
          mx1 = fmaxf(mx1, fmaxf(__uint_as_float(v[k + 2]), __uint_as_float(v[k + 3])));
          mx2 = fmaxf(mx2, fmaxf(__uint_as_float(v[k + 4]), __uint_as_float(v[k + 5])));
          mx3 = fmaxf(mx3, fmaxf(__uint_as_float(v[k + 6]), __uint_as_float(v[k + 7])));
        }
        const float m_new = fmaxf(m, fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * a.scale_log2);   // scale > 0: the maximum commutes with it
        // tensor-memory loads and stores are warp-wide: the warp moves its maxima together, as soon as one of
        // its rows has outgrown its own by the step (a row that has not may follow the true maximum just as well)
        const bool move = __any_sync(0xffffffffu, m_new > m + RESCALE_STEP);
        // P(i) goes where P(i - 1) lay: the product that read it must be complete
        if (h == 0 && i > 0 && !wait_pv(i - 1)) {
          ok = false;
          break;
        }
        if (move) {
          const float corr = fast_exp2(m - (m_new == -INFINITY ? 0.0f : m_new));   // m = -inf gives 0
          m = m_new;
          l *= corr;
          if (h > 0) {   // this block's first piece: its partial sums, and its probabilities where this thread wrote them
            l0 *= corr, l1 *= corr, l2 *= corr, l3 *= corr;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const uint32_t at = p_row + ((uint32_t)(c << 4) ^ p_xor);
              uint32_t w[4];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 pair = *reinterpret_cast<const __nv_bfloat162*>(&w[e]);
                w[e] = pack_bf16(__low2float(pair) * corr, __high2float(pair) * corr);
              }
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
            }
          }
          if (i > 0) {     // O = O * corr in tensor memory, between two products (the one before is complete: see above)
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
            tmem_wait_stores();
          }
        }
        const float m_use = m == -INFINITY ? 0.0f : m;
        // probabilities into shared memory as the A operand of P V (sub-tile h of 64 keys); the row's sum
        // in four independent partial sums
#pragma unroll
        for (int c = 0; c < S_PIECE / 8; ++c) {
          uint32_t packed[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = fast_exp2(fmaf(__uint_as_float(v[c * 8 + 2 * e]), a.scale_log2, -m_use));
            const float p1 = fast_exp2(fmaf(__uint_as_float(v[c * 8 + 2 * e + 1]), a.scale_log2, -m_use));
            if (e == 0) l0 += p0 + p1;
            else if (e == 1) l1 += p0 + p1;
            else if (e == 2) l2 += p0 + p1;
            else l3 += p0 + p1;
            packed[e] = pack_bf16(p0, p1);
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p_row + h * SUB + ((uint32_t)(c << 4) ^ p_xor)),
                       "r"(packed[0]), "r"(packed[1]), "r"(packed[2]), "r"(packed[3]) : "memory");
        }
      }
      if (!ok) break;
      l += (l0 + l1) + (l2 + l3);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&p_full[g]);
    }
    if (ok && my_n > 0) ok = wait_pv(my_n - 1) && !*abort_flag;
    if (!ok) {
      *abort_flag = 1;
      atomicCAS(a.error_word, 0, ERR_SOFTMAX);
    }
    // ---- every thread finishes its own row: O / l out of tensor memory, rounded to bfloat16, 64 bytes
    // at a time.  Heads that share a key/value head lie side by side in a token's output row, as their
    // rows do in the tile.  (The loads are warp-wide, so rows without an output still take part.)
    if (ok && my_n > 0) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int token = row_valid ? R / group : 0, head = row_valid ? kvh * group + R % group : 0;
      // the sink joins the sum, taken against the same maximum (far above it the sum is infinite, the row zero)
      if (extras.sink && row_valid) l += exp2f(sink_log2(extras, head) - m);
      const float inv = l > 0.0f ? (row_valid ? head_gate<__nv_bfloat16>(extras, q_start + token, head) : 1.0f) / l : 0.0f;
      uint4* dst = reinterpret_cast<uint4*>(a.out + ((long long)(q_start + token) * a.q_heads + head) * D);
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t t[32];
        tmem_load32_nowait(o_addr + c0, t);
        tmem_wait_loads();
        if (row_valid) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            dst[c0 / 8 + c] = make_uint4(pack_bf16(__uint_as_float(t[8 * c]) * inv, __uint_as_float(t[8 * c + 1]) * inv),
                                         pack_bf16(__uint_as_float(t[8 * c + 2]) * inv, __uint_as_float(t[8 * c + 3]) * inv),
                                         pack_bf16(__uint_as_float(t[8 * c + 4]) * inv, __uint_as_float(t[8 * c + 5]) * inv),
                                         pack_bf16(__uint_as_float(t[8 * c + 6]) * inv, __uint_as_float(t[8 * c + 7]) * inv));
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

}  // namespace

extern "C" int llm_cache8_attention_prompt_rows() { return BLOCK_ROWS; }

// The tiles of llm_step_maps with tile_rows = llm_cache8_attention_prompt_rows() (entries of -1 return at once).  chunk, sink, gate and
// gate_stride (elements): `AttentionExtras`; 0 and null: none.
extern "C" int llm_cache8_attention_prompt(const void* q, void* out, const Cache8* cache, const int32_t* seq_q_start,
                                           const int32_t* seq_q_len, const int32_t* seq_kv_len, const int32_t* tile_seq,
                                           const int32_t* tile_index, int n_tiles, int q_heads, float scale, int window, int chunk,
                                           const float* sink, const void* gate, long long gate_stride, int* error_word,
                                           cudaStream_t stream) {
  if (n_tiles <= 0) return 0;
  const Cache8& c = *cache;
  if (c.head_dim != D || c.kv_heads <= 0 || q_heads <= 0 || q_heads % c.kv_heads || c.page_tokens <= 0 || c.page_tokens % SCALE_TOKENS ||
      n_tiles > 65535 || !(scale > 0.0f))
    return ERR_BAD_SIZE;
  const uintptr_t all = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(c.k) |
                        reinterpret_cast<uintptr_t>(c.v) | (uintptr_t)c.page_stride;
  if (all & 15) return ERR_BAD_ALIGN;
  static bool configured = false;
  if (!configured) {
    if (cudaFuncSetAttribute(cache8_prompt_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(cache8_prompt_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES) != cudaSuccess)
      return launch_status();
    configured = true;
  }
  const AttnArgs a{reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<__nv_bfloat16*>(out), c, seq_q_start, seq_q_len,
                   seq_kv_len, tile_seq, tile_index, q_heads, scale * 1.4426950408889634f, window,
                   AttentionExtras{chunk, sink, gate, gate_stride}, error_word};
  launch_kernel(window > 0 || chunk > 0 || sink || gate ? cache8_prompt_kernel<true> : cache8_prompt_kernel<false>,
                dim3(c.kv_heads, n_tiles), NUM_THREADS, SMEM_BYTES, stream, a);
  return launch_status();
}
