// Softmax attention of prompt portions over a cache of e4m3 codes (cache8.cuh) on the Blackwell tensor cores: what
// attention_tcgen05.cu is to a bfloat16 cache, for requests with more than 16 packed rows (tokens x query heads of one key/value
// head).  Nothing of cuongvng/bare-cuda-4gib's [heads, T, keys] score buffer exists (engine/kernels/attention_qk.cu:49-68,
// softmax.cu:28-42, attention_av.cu:24-44).
//
//   s[k] = scale * 2^e_K(k) * (q . K_k)     p = softmax over the visible k     out = sum_k p[k] 2^e_V(k) V_k
//
// One thread block = two tiles of 128 packed rows of one request and one key/value head, which share every key and value block of 128
// positions.  Warps:
//   loader (1)     copies a key block's codes, as they lie in the request's pages, into shared memory with TMA (one tensor map over the cache's
//                  pool, a box per piece of a page), and hands the block's scales to the softmax;
//   converters (4) write the value codes as halves (which hold e4m3 exactly, two a conversion) into 128-byte-swizzled tiles;
//   MMA issuers (2, one a tile)  S_g = Q_g K^T (M 128, N 64, twice a key block) with the keys as the codes they are: an 8-bit product.  Q_g is the sum of two
//                  e4m3 tiles, which together hold a bfloat16's eight bits exactly (but for entries below 2^-9 of their row's largest, which are off by at most 2^-17 of it), times a power of
//                  two of the row's own; two products at twice the rate of one in 16 bits, and no key is ever converted.
//                  O_g (+)= P_g V in halves of 64 keys, each as soon as its half of P is there, with P_g as the operand in tensor memory and V as it
//                  lies ([key][channel], MN-major): P never goes through shared memory, whose bandwidth bounds a block that has it there;
//   softmax (8)    a group of four warps per tile, one thread per row.  First it stages Q_g.  Then, per half of 64 keys: read the row of S, mask,
//                  running maximum and sum in float32 (base 2), write P as halves back into tensor memory.
// The scales cost the softmax nothing but their constants: the keys' joins the factor of 16 scores, and a weight goes into P together with the
// scale of its values: P = 2^(s + e_V - m + 7) with m the running maximum of s + e_V, while the sum takes P 2^(-e_V - 7).  So a half of P is relative to
// what the row's keys can add to its output, and O needs no factor of its own but the 2^-7 at the end.  The 2^7 is for rows of which one token takes
// most of the weight: weights keep a half's eleven bits down to 2^-21 of the largest (15 nats below it),
// have an absolute step of 2^-31 of it from there on, and are lost from O below 2^-32.  Of a block whose values are all below 2^-60 of the
// largest so far (one of zeros, say, whose scale is the least one) such a P may leave nothing to take a sum from: for those the sum takes 2^(s - m)
// itself, a second exponential, where the maximum is moved (2 % for the code's presence; behind the first ones 4 %, in a loop of its own 8 %).
// Larger values that are hidden from a row do not matter to it: the second way is right for any values.
// m follows the true maximum only when that has grown by more than 2^8 (a half reaches 2^15), so O is rescaled rarely.
// A half of P takes the columns of the scores it was made of (S 2 x 128, O 2 x head size columns of the 512), and the next key block's half of S is
// issued when P has been read, while the softmax is at the other half: it waits for no product.
// Few tiles (a question behind a long text): the key blocks are split among the blocks of a cluster, each with a softmax of its own; their
// states are merged in index order through distributed shared memory.
// A NaN scale (a block that was given a NaN) makes NaN of its 16 scores before hidden ones are replaced, so that only rows that see
// the block get it; values are finite always, and behind the request's last key, or where no page is held, written as zeros.
// Every mbarrier wait is bounded: on a timeout the thread sets the error word, all roles leave their loops, tensor memory is
// released and the block returns.
// One B200: a prompt of 2,048 tokens (32 / 4 heads of 64) 43.9 us (over a bfloat16 cache 41.3), 2,048 tokens behind 2,048 (32 heads of 128) 117 us
// (0.88 PFLOP/s; 136), 61 tokens behind 3,001 (32 / 8 heads of 128) 20.6 us (66).  What bounds it: a key block takes about 4,300 cycles for 256 rows,
// of which the exponential unit is busy 1,540 and the tensor cores 1,000 to 2,000; the softmax warps (two a scheduler) wait for tensor-memory loads
// and for their own chains of dependent instructions.  A block's start (queries staged: 7,000 cycles) and the merge of a cluster (9,000) weigh most
// where there are few keys a block.

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
constexpr int BM = 128;          // packed rows per tile (one softmax group)
constexpr int TILES = 2;         // tiles per block: both read every key and value tile
constexpr int BLOCK_ROWS = TILES * BM;
constexpr int BN = 128;          // keys per block
constexpr int CODES = BN * D;    // bytes of a key tile, of a value tile as codes, and of each part of a tile's queries
constexpr int SUB = 128 * 128;   // bytes of a [128 keys x 64 halves] swizzled sub-tile
constexpr int VALUES = D / 64 * SUB;     // bytes of a value tile as halves
// what is in flight (as shared memory allows): key tiles, value tiles as codes, value tiles as halves
constexpr int K_SLOTS = 4, C_SLOTS = HEAD_DIM == 64 ? 4 : 2, V_SLOTS = HEAD_DIM == 64 ? 4 : 2;
constexpr int SOFTMAX_THREADS = 128 * TILES, CONVERT_THREADS = 128;
constexpr int CONVERT_WARP = SOFTMAX_THREADS / 32, MMA_WARP = CONVERT_WARP + CONVERT_THREADS / 32, LOADER_WARP = MMA_WARP + TILES;
constexpr int NUM_THREADS = (LOADER_WARP + 1) * 32;   // warps 0-7 softmax, 8-11 converters, 12 and 13 MMA (one a tile), 14 loader
constexpr int GROUP_THREADS = 128;
constexpr int S_PIECE = 64;      // columns of S a softmax thread holds in registers at a time
constexpr int TMEM_COLS = 512, O_COL = TILES * BN;
constexpr unsigned long long WAIT_LIMIT_NS = 1000000000ull;
constexpr float RESCALE_STEP = 8.0f;
constexpr int HEADROOM = 7;      // with the step above, what a half can hold over one: 2^15
constexpr float P_UNIT = 1.0f / (1 << HEADROOM);
static_assert(HEADROOM <= 126 - SCALE_MOST, "the sum takes 2^(-e_V - HEADROOM)");
// What the factor of 16 scores is kept within: at 0 a hidden score (-inf) would be no longer hidden (2^-126 more changes none above 2^-102, and
// ones below make nothing of any score), and an infinite factor times a score of zero would be no number.
constexpr float LEAST_FACTOR = 1.17549435e-38f, MOST_FACTOR = 3.40282347e38f;
constexpr int CHUNKS = D / 16;              // 16-byte chunks of a key's codes; also how many of them a converter thread takes of a tile
constexpr int BLOCKS = BN / SCALE_TOKENS;   // scale blocks of a key block
constexpr int MAX_SPLITS = 8;               // blocks that may share a tile's keys
constexpr int KNOWN = 8;                    // key blocks whose scales are kept (a key tile's slot is free again at most five blocks on)
constexpr int VALUE_RANGE = 60;             // how far below the largest exponent of a value scale a sum still takes its part from P (base 2)
constexpr int STATE = D + 4;                // floats of a row's state in a merge: D sums, the maximum, the sum
constexpr size_t TILES_BYTES = (size_t)(TILES * 2 + K_SLOTS + C_SLOTS) * CODES + (size_t)V_SLOTS * VALUES;
static_assert((size_t)BLOCK_ROWS * STATE * 4 <= TILES_BYTES, "the states of a merge lie over the tiles");
// A key block's scales as the softmax takes them, 16 positions each.
struct Scales {
  float key[BLOCKS];       // 2^e_K (1 where it is lost)
  float value[BLOCKS];     // e_V
  float back[BLOCKS];      // 2^(-e_V - HEADROOM); 0 where the sum takes its part another way
  uint32_t special, unused[3];   // bits b, 8 + b, 16 + b: scale block b has no number as its keys' scale, has no page, has values far below others
};

// barriers (two to a slot, 14 of the groups, one to a block of scales), scales, rows' exponents, what is held, two words; 16 for alignment
constexpr size_t BOOK_BYTES = 8 * (2 * (K_SLOTS + C_SLOTS + V_SLOTS) + 14 + KNOWN) + 16 + KNOWN * sizeof(Scales) + 4 * (BLOCK_ROWS + C_SLOTS + 2);
constexpr size_t SMEM_BYTES = TILES_BYTES + BOOK_BYTES;
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

// Byte offset of the 16-byte chunk `chunk` (0..7) of row `row` inside a [rows x 64 halves] sub-tile
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
__device__ __forceinline__ uint32_t codes_swizzled(int row, int chunk) {
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

// The same for tiles of codes, whose rows are D bytes: 128-byte swizzle, or 64-byte swizzle with 512 bytes between 8-row groups.
__device__ __forceinline__ uint64_t smem_desc_codes(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(8 * D >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)(D == 128 ? 2 : 4) << 61;
  return d;
}

// float32 accumulator, half operands (kind::f16) or e4m3 ones (kind::f8f6f4), A K-major; B K-major or (b_mn = 1) MN-major.
__host__ __device__ constexpr uint32_t instr_desc(int m, int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_codes(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
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
__device__ __forceinline__ void tmem_load16_nowait(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
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
// Maxima that keep a NaN.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// 2^x for both of a pair without the exponential unit, which takes eight cycles a warp and is what the softmax would wait for: x = n + f with
// n the nearest whole number (found by adding 1.5 * 2^23), 2^f by a polynomial that was fitted to it on [-1/2, 1/2] for the least
// relative error (2.9e-6) with 1 at 0, n added to its exponent.  Up to x = -127: zero, as that exponent says of a one.  A NaN becomes zero too:
// the row's maximum keeps it.  One pair of four goes this way: the 7b portion below 122 -> 117 us.
__device__ __forceinline__ void exp2_by_products(uint64_t x, float& p0, float& p1) {
  float a, b;
  unpair(x, a, b);
  a = fmaxf(a, -127.0f), b = fmaxf(b, -127.0f);
  x = pair(a, b);
  const uint64_t big = pair(12582912.0f, 12582912.0f), minus_big = pair(-12582912.0f, -12582912.0f), minus_one = pair(-1.0f, -1.0f);
  const uint64_t r = add2(x, big), f = fma2(add2(r, minus_big), minus_one, x);
  uint64_t p = fma2(f, pair(0.009582576f, 0.009582576f), pair(0.05590683f, 0.05590683f));
  p = fma2(p, f, pair(0.24024107f, 0.24024107f));
  p = fma2(p, f, pair(0.6931241f, 0.6931241f));
  p = fma2(p, f, pair(1.0f, 1.0f));
  float n0, n1;
  unpair(r, n0, n1);
  unpair(p, p0, p1);
  p0 = __int_as_float(__float_as_int(p0) + (__float_as_int(n0) << 23));
  p1 = __int_as_float(__float_as_int(p1) + (__float_as_int(n1) << 23));
}
// Four codes as four halves.
__device__ __forceinline__ void halves(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(codes));
}
// The factor of 16 scores.
__device__ __forceinline__ float score_factor(float of_row, float of_keys) { return fminf(fmaf(of_row, of_keys, LEAST_FACTOR), MOST_FACTOR); }
// Two numbers as two e4m3 codes.
__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
// Two halves less the two numbers of `codes`, as codes.
__device__ __forceinline__ uint32_t rest_codes2(uint32_t numbers, uint32_t codes) {
  uint16_t d;
  asm("{\n\t.reg .b32 h;\n\tcvt.rn.f16x2.e4m3x2 h, %2;\n\tsub.rn.f16x2 h, %1, h;\n\tcvt.rn.satfinite.e4m3x2.f16x2 %0, h;\n\t}"
      : "=h"(d) : "r"(numbers), "h"((uint16_t)codes));
  return d;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
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
  uint8_t* q_smem = smem;                              // [TILES][2]: the queries' two parts
  uint8_t* k_ring = q_smem + TILES * 2 * CODES;        // [K_SLOTS]
  uint8_t* c_ring = k_ring + K_SLOTS * CODES;          // [C_SLOTS]: values as codes
  uint8_t* v_ring = c_ring + C_SLOTS * CODES;          // [V_SLOTS]: values as halves
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + TILES_BYTES);
  uint64_t* k_full = bars;                  // [K_SLOTS] loader -> MMA: the slot's keys have landed
  uint64_t* k_empty = k_full + K_SLOTS;     // [K_SLOTS] both MMA issuers (commit) -> loader
  uint64_t* c_full = k_empty + K_SLOTS;     // [C_SLOTS] loader -> converters: the slot's value codes have landed
  uint64_t* c_empty = c_full + C_SLOTS;     // [C_SLOTS] converters -> loader
  uint64_t* v_full = c_empty + C_SLOTS;     // [V_SLOTS] converters -> MMA: the slot's values are written
  uint64_t* v_empty = v_full + V_SLOTS;     // [V_SLOTS] both MMA issuers (commit) -> converters
  uint64_t* q_full = v_empty + V_SLOTS;     // [2] softmax group -> MMA: Q_g staged
  uint64_t* s_full = q_full + 2;            // [2][2] MMA (commit) -> softmax, per group and half of 64 keys
  uint64_t* p_full = s_full + 4;            // [2][2] softmax -> MMA: half h of P written
  uint64_t* pv_done = p_full + 4;           // [2][2] MMA (commit) -> softmax, MMA: the product with half h is complete
  uint64_t* known = pv_done + 4;            // [KNOWN] loader -> MMA (-> softmax, with s_full): a key block's scales
  Scales* scales = reinterpret_cast<Scales*>((reinterpret_cast<uintptr_t>(known + KNOWN) + 15) & ~uintptr_t(15));   // [KNOWN]
  int* q_exponent = reinterpret_cast<int*>(scales + KNOWN);     // [BLOCK_ROWS] of the power of two taken out of a row of Q
  uint32_t* held = reinterpret_cast<uint32_t*>(q_exponent + BLOCK_ROWS);   // [C_SLOTS] bit b: there are values for scale block b
  uint32_t* tmem_slot = held + C_SLOTS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // ---- what this block works on (uniform across the cluster).  The step's lists are there before its kernels start, so they may
  // be read ahead of pdl_wait().  Blocks are handed out with x fastest: all key/value heads of the latest tile first (it sees
  // the most keys), then of the tile before it, ...
  const int tile = gridDim.y - 1 - blockIdx.y, kvh = blockIdx.x;
  const int seq = a.lists.tile_seq[tile];
  if (seq < 0) {              // the end of the list; the blocks of its first entry stay for the kernels before (a kernel may not end ahead of them),
    if (tile == 0) pdl_wait();  // the others hold up no block that has work
    return;
  }
  if (smem_u32(smem) & 1023) {   // never seen; refuse rather than compute with a broken layout
    if (threadIdx.x == 0) atomicCAS(a.error_word, 0, ERR_LAYOUT);
    return;
  }
  const int group = a.q_heads / a.cache.kv_heads;
  const int q_start = a.lists.seq_q_start[seq], q_len = a.lists.seq_q_len[seq], kv_len = a.lists.seq_kv_len[seq];
  const int row0 = a.lists.tile_index[tile] * BLOCK_ROWS, n_rows = q_len * group, pos0 = kv_len - q_len;
  if (row0 >= n_rows) {      // (rows that the step does not have)
    pdl_wait();
    return;
  }
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
    for (int s = 0; s < K_SLOTS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], TILES);
    }
    for (int s = 0; s < C_SLOTS; ++s) {
      mbar_init(&c_full[s], 1);
      mbar_init(&c_empty[s], CONVERT_THREADS / 32);
    }
    for (int s = 0; s < V_SLOTS; ++s) {
      mbar_init(&v_full[s], CONVERT_THREADS / 32);
      mbar_init(&v_empty[s], TILES);
    }
    for (int s = 0; s < KNOWN; ++s) mbar_init(&known[s], 1);
    for (int b = 0; b < 2; ++b) mbar_init(&q_full[b], GROUP_THREADS);
    for (int b = 0; b < 4; ++b) {
      mbar_init(&s_full[b], 2);        // the product, the issuer (which has seen the scales)
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
    for (int jj = 0; jj < n_kb; ++jj) {
      const int from_slot = jj % C_SLOTS, slot = jj % V_SLOTS, use = jj / V_SLOTS;
      ok = mbar_wait(&c_full[from_slot], (uint32_t)(jj / C_SLOTS) & 1u, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint4 raw[CHUNKS];
      const uint32_t from = smem_u32(c_ring) + from_slot * CODES, there = held[from_slot];
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[i].x), "=r"(raw[i].y), "=r"(raw[i].z), "=r"(raw[i].w) : "r"(from + codes_swizzled(row_in + i * STEP, chunk)) : "memory");
      const int behind = kv_len - (kb_lo + jj) * BN;       // rows from here on lie behind the request's last key
      if (behind < BN || there != (1u << BLOCKS) - 1u) {   // what lies where there are no values may be anything, and zero times NaN is not zero
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          const int row = row_in + i * STEP;
          if (row >= behind || !((there >> (row / SCALE_TOKENS)) & 1u)) raw[i] = make_uint4(0, 0, 0, 0);
        }
      }
      ok = use == 0 || mbar_wait(&v_empty[slot], (uint32_t)(use - 1) & 1u, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint32_t to = smem_u32(v_ring) + slot * VALUES + (chunk >> 2) * SUB;
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        const int row = row_in + i * STEP, first = (chunk & 3) * 2;
        uint32_t w[8];
        halves(raw[i].x, w[0], w[1]);
        halves(raw[i].y, w[2], w[3]);
        halves(raw[i].z, w[4], w[5]);
        halves(raw[i].w, w[6], w[7]);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + swizzled(row, first)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + swizzled(row, first + 1)), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&c_empty[from_slot]);      // (here, where every lane's loads of the codes have arrived, not where they were asked for)
        mbar_arrive(&v_full[slot]);
      }
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
    const int per_piece = a.box_rows / SCALE_TOKENS;
    const bool leads = lane < BLOCKS && lane % per_piece == 0;      // a piece of a page is its first scale block's lane's to copy
    bool ok = true;
    int k_issued = 0, c_issued = 0;
    auto copy = [&](uint64_t* full, uint8_t* slot, const Place& p, long long row0, uint32_t copies) {
      if (lane == 0) mbar_expect_tx(full, copies * a.box_rows * D);   // also the one arrival
      __syncwarp();
      if (leads && p.row >= 0) tma_load_2d(smem_u32(slot) + lane * SCALE_TOKENS * D, &pool_map, full, 0, (int)(p.row + row0));
    };
    Place now = place(0, find_page(0));
    int page = -1, most = SCALE_LEAST;        // the largest exponent of a value scale so far
    for (int jj = 0; jj < n_kb; ++jj) {
      int ev = now.row >= 0 ? max(exponent_of(now.v_scale), SCALE_LEAST) : SCALE_LEAST;      // (a scale that nothing has written is zero)
      most = max(most, __reduce_max_sync(0xffffffffu, ev));
      if (now.row < 0) ev = most;
      const bool far = ev < most - VALUE_RANGE;
      const uint32_t there = __ballot_sync(0xffffffffu, now.row >= 0), copies = __popc(__ballot_sync(0xffffffffu, leads && now.row >= 0));
      const int ks = jj % K_SLOTS, cs = jj % C_SLOTS;
      ok = jj < K_SLOTS || mbar_wait(&k_empty[ks], (uint32_t)(jj / K_SLOTS - 1) & 1u, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      copy(&k_full[ks], k_ring + ks * CODES, now, a.k_row0, copies);
      k_issued = jj + 1;
      ok = jj < C_SLOTS || mbar_wait(&c_empty[cs], (uint32_t)(jj / C_SLOTS - 1) & 1u, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) held[cs] = there;
      copy(&c_full[cs], c_ring + cs * CODES, now, a.v_row0, copies);
      c_issued = jj + 1;
      if (jj == 0) page = find_page(1);
      const Place next = place(jj + 1, page);
      page = find_page(jj + 2);
      // the scales, while the codes are on their way
      const bool lost = isnan(now.k_scale);
      Scales* to = scales + jj % KNOWN;
      if (lane < BLOCKS) {
        to->key[lane] = now.row >= 0 && !lost ? fmaxf(now.k_scale, power_of_two(SCALE_LEAST)) : 1.0f;
        to->value[lane] = (float)ev;
        to->back[lane] = far ? 0.0f : power_of_two(-ev - HEADROOM);
      }
      const uint32_t all_far = __ballot_sync(0xffffffffu, far);
      const uint32_t all_lost = __ballot_sync(0xffffffffu, lost && now.row >= 0);
      const uint32_t all_absent = __ballot_sync(0xffffffffu, lane < BLOCKS && now.row < 0 && (kb_lo + jj) * BN + lane * SCALE_TOKENS < kv_len);
      if (lane == 0) to->special = all_lost | all_absent << 8 | all_far << 16;
      __syncwarp();
      if (lane == 0) mbar_arrive(&known[jj % KNOWN]);
      now = next;
    }
    if (!ok) {
      if (lane == 0) {
        *abort_flag = 1;
        atomicCAS(a.error_word, 0, ERR_LOADER);
        // this block's copies in flight land before it leaves (the waits of the others end at the flag)
        volatile int never = 0;
        for (int n = max(0, k_issued - K_SLOTS); n < k_issued; ++n) mbar_wait(&k_full[n % K_SLOTS], (uint32_t)(n / K_SLOTS) & 1u, &never);
        for (int n = max(0, c_issued - C_SLOTS); n < c_issued; ++n) mbar_wait(&c_full[n % C_SLOTS], (uint32_t)(n / C_SLOTS) & 1u, &never);
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
      const uint64_t q_desc = smem_desc_codes(smem_u32(q_smem) + g * 2 * CODES);
      bool ok = true;
      auto keys_landed = [&](int jj) { return mbar_wait(&k_full[jj % K_SLOTS], (uint32_t)(jj / K_SLOTS) & 1u, abort_flag); };
      auto values_landed = [&](int jj) { return mbar_wait(&v_full[jj % V_SLOTS], (uint32_t)(jj / V_SLOTS) & 1u, abort_flag); };
      // half h of S_g = Q_g K(jj)^T
      auto issue_s = [&](int jj, int h) {
        const int slot = jj % K_SLOTS, i = jj - lo;
        ok = ok && (h > 0 || keys_landed(jj)) && (i > 0 ? mbar_wait(&pv_done[g * 2 + h], (uint32_t)(i - 1) & 1u, abort_flag)   // P(i - 1) has been read
                                                        : h > 0 || mbar_wait(&q_full[g], 0, abort_flag));
        if (!ok) return;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t k_desc = smem_desc_codes(smem_u32(k_ring) + slot * CODES + h * S_PIECE * D);
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            umma_codes(s_tmem + h * S_PIECE, q_desc + (part * CODES >> 4) + 2 * k, k_desc + 2 * k, idesc_s, (part > 0 || k > 0) ? 1u : 0u);
        umma_commit(&s_full[g * 2 + h]);
        if (h == 1) umma_commit(&k_empty[slot]);
        // the group reads the block's scales behind s_full
        ok = ok && (h > 0 || mbar_wait(&known[jj % KNOWN], (uint32_t)(jj / KNOWN) & 1u, abort_flag));
        mbar_arrive(&s_full[g * 2 + h]);
      };
      // O_g (+)= half h of P_g V(jj): the group's O accumulates in tensor memory over its key blocks
      auto issue_pv = [&](int jj, int h) {
        const int slot = jj % V_SLOTS, i = jj - lo;
        ok = ok && (h > 0 || values_landed(jj)) && mbar_wait(&p_full[g * 2 + h], (uint32_t)i & 1u, abort_flag);
        if (!ok) return;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t v_desc = smem_desc_sw128(smem_u32(v_ring) + slot * VALUES, SUB);
#pragma unroll
        for (int kk = 0; kk < S_PIECE / 16; ++kk)
          umma_ts(o_tmem, s_tmem + h * S_PIECE + kk * 8, v_desc + (uint64_t)((h * (S_PIECE / 16) + kk) * 2048 >> 4), idesc_o,
                  (kk > 0 || h > 0 || i > 0) ? 1u : 0u);
        umma_commit(&pv_done[g * 2 + h]);
        if (h == 1) umma_commit(&v_empty[slot]);
      };
      auto pass = [&](int jj) {       // a key block that only the other tile reads
        ok = ok && keys_landed(jj);
        if (ok) mbar_arrive(&k_empty[jj % K_SLOTS]);
        ok = ok && values_landed(jj);
        if (ok) mbar_arrive(&v_empty[jj % V_SLOTS]);
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
    // D / 8 threads to a row of Q, so that the loads are whole lines; where a row lies, and its power of two, the row's own thread knows
    constexpr int LANES = D / 8, ROWS = 32 / LANES;          // of a load of the warp
    constexpr int BATCH = 4;                                 // loads on their way at once
    const long long my_at = row_valid ? ((long long)(q_start + token) * a.q_heads + head) * D : -1;
#pragma unroll 1
    for (int batch = 0; batch < 32 / ROWS / BATCH; ++batch) {
      uint4 raw[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const long long at = __shfl_sync(0xffffffffu, my_at, (batch * BATCH + i) * ROWS + lane / LANES);
        raw[i] = make_uint4(0, 0, 0, 0);
        if (at >= 0) raw[i] = __ldg(reinterpret_cast<const uint4*>(a.q + at) + lane % LANES);
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int in_tile = (warp & 3) * 32 + (batch * BATCH + i) * ROWS + lane / LANES, c = lane % LANES;
        const uint32_t* pairs = reinterpret_cast<const uint32_t*>(&raw[i]);
        uint32_t most = 0;                     // of the magnitudes' bits, which are in the order of the numbers
#pragma unroll
        for (int k = 0; k < 4; ++k) most = max_u16x2(most, pairs[k] & 0x7fff7fffu);
#pragma unroll
        for (int by = 1; by < LANES; by <<= 1) most = max_u16x2(most, __shfl_xor_sync(0xffffffffu, most, by));
        most = max(most & 0xffffu, most >> 16);
        const int e = most > 0 ? min(max((int)(most >> 7) - 127 - 7, -100), 119) : 0;     // the largest entry to [2^7, 2^8)
        const float down = most < 0x7f80u ? power_of_two(-e) : __int_as_float(0x7fc00000);   // (codes have no infinity: such a row becomes NaN)
        uint32_t part[2][2];
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          uint32_t first[2], rest[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float x = __uint_as_float(pairs[k + u] << 16) * down, y = __uint_as_float(pairs[k + u] & 0xffff0000u) * down;
            first[u] = codes2(x, y);
            rest[u] = rest_codes2(pack_half(x, y), first[u]);      // (halves hold both numbers exactly)
          }
          part[0][k >> 1] = first[0] | first[1] << 16;
          part[1][k >> 1] = rest[0] | rest[1] << 16;
        }
        const uint32_t to = smem_u32(q_smem) + g * 2 * CODES + codes_swizzled(in_tile, c >> 1) + (c & 1) * 8;
        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(part[0][0]), "r"(part[0][1]) : "memory");
        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + CODES), "r"(part[1][0]), "r"(part[1][1]) : "memory");
        if (c == 0) q_exponent[g * BM + in_tile] = e;
      }
    }
    __syncwarp();
    const float factor = a.scale_log2 * power_of_two(q_exponent[g * BM + r]);       // (this warp wrote it)
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mbar_arrive(&q_full[g]);
    const int row_pos = row_valid ? pos0 + token : -1;
    const uint32_t s_addr = lane_addr + g * BN;
    const int row_lo = first_visible_key(row_pos, window, extras.chunk);
    const int tile_min_pos = g ? g_min_pos[1] : g_min_pos[0];
    const int tile_max_lo = first_visible_key(g ? g_max_pos[1] : g_max_pos[0], window, extras.chunk);   // from here on no row's bound hides a key
    // the product with half h of this group's block k is complete
    auto wait_pv = [&](int k, int h) { return mbar_wait(&pv_done[g * 2 + h], (uint32_t)k & 1u, abort_flag); };
    uint64_t l2 = 0;         // the row's sum, in two parts
    bool ok = true;
    for (int i = 0; i < my_n && ok; ++i) {
      const int jj = my_lo + i - kb_lo, key0 = (my_lo + i) * BN;
      const Scales* of_block = scales + jj % KNOWN;
      const bool all_visible = key0 + BN - 1 <= tile_min_pos && (!EXTRAS || key0 >= tile_max_lo);
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        ok = ok && mbar_wait(&s_full[g * 2 + h], (uint32_t)i & 1u, abort_flag) && (h > 0 || !*abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t v[S_PIECE];
#pragma unroll
        for (int k = 0; k < S_PIECE; k += 32) tmem_load32_nowait(s_addr + h * S_PIECE + k, v + k);
        tmem_wait_loads();
        const uint32_t special = of_block->special >> (h * 4);
        float limit = m + RESCALE_STEP;      // what a row's maximum may grow to before its sums follow
        if (special & 0x0f0f0fu) {
          if (special & 0x0f0000u) limit = __int_as_float(0x7fc00000);      // (they follow in any case)
#pragma unroll
          for (int k = 0; k < S_PIECE; ++k) {
            if ((special >> (k / SCALE_TOKENS)) & 1u) v[k] = 0x7fc00000u;
            if ((special >> (8 + k / SCALE_TOKENS)) & 1u) v[k] = 0xff800000u;
          }
        }
        if (!all_visible) {
#pragma unroll
          for (int k = 0; k < S_PIECE; ++k) {
            const int key = key0 + h * S_PIECE + k;
            const bool visible = key <= row_pos && (!EXTRAS || key >= row_lo);
            if (!visible) v[k] = 0xff800000u;   // -inf: probability 0
          }
        }
        // The exponentials are taken against the maximum so far while the scores' own is being found, which needs them only when it has
        // outgrown the other by the step: then they are taken again (twice or so for a row of many blocks).
        for (bool settled = false;; settled = true) {
          const float m_use = m == -INFINITY ? 0.0f : m - HEADROOM;
          float m_new = m;
          uint64_t sum = l2;
          uint32_t packed[16];
#pragma unroll
          for (int j = 0; j < S_PIECE / SCALE_TOKENS; ++j) {
            const uint32_t* w = v + j * SCALE_TOKENS;
            const float c = score_factor(factor, of_block->key[h * 4 + j]), ev = of_block->value[h * 4 + j], back = of_block->back[h * 4 + j];
            const uint64_t c2 = pair(c, c), shift2 = pair(ev - m_use, ev - m_use);
            uint64_t part = 0;
#pragma unroll
            for (int k = 0; k < SCALE_TOKENS; k += 2) {
              const uint64_t x = fma2(pair(__uint_as_float(w[k]), __uint_as_float(w[k + 1])), c2, shift2);
              float p0, p1;
              if (k % 8 == 4) {
                exp2_by_products(x, p0, p1);
              } else {
                unpair(x, p0, p1);
                p0 = fast_exp2(p0), p1 = fast_exp2(p1);
              }
              part = k == 0 ? pair(p0, p1) : add2(part, pair(p0, p1));
              packed[(j & 1) * 8 + k / 2] = pack_half(p0, p1);
            }
            sum = fma2(part, pair(back, back), sum);
            float even = __uint_as_float(w[0]), odd = __uint_as_float(w[1]);
#pragma unroll
            for (int k = 2; k < SCALE_TOKENS - 2; k += 4) {
              even = max3(even, __uint_as_float(w[k]), __uint_as_float(w[k + 1]));
              odd = max3(odd, __uint_as_float(w[k + 2]), __uint_as_float(w[k + 3]));
            }
            const float most = max3(max2(even, odd), __uint_as_float(w[SCALE_TOKENS - 2]), __uint_as_float(w[SCALE_TOKENS - 1]));
            m_new = max2(m_new, fmaf(most, c, ev));   // c > 0: the maximum commutes with it
            if (j & 1) tmem_store16(s_addr + h * S_PIECE + (j >> 1) * 16, packed);      // over the scores that they were made of
          }
          // tensor-memory loads and stores are warp-wide: the warp moves its maxima together, as soon as one of
          // its rows has outgrown its own by the step (a row that has not may follow the true maximum just as well).  A row that
          // sees a score that is no number has no number as its maximum either, and from here on as its sum.
          if (settled || !__any_sync(0xffffffffu, !(m_new <= limit))) {
            l2 = sum;
            break;
          }
          const float down = m - (m_new == -INFINITY ? 0.0f : m_new), half_way = fast_exp2(0.5f * down), corr = fast_exp2(down);   // m = -inf gives 0
          m = m_new;
          l2 = fma2(fma2(l2, pair(half_way, half_way), 0), pair(half_way, half_way), 0);
          const uint32_t far = of_block->special >> (16 + h * 4);
          if (far & 0x0fu) {        // the shares of blocks whose values are far below others
            const float m_use = m == -INFINITY ? 0.0f : m;
            float share = 0.0f;
#pragma unroll
            for (int k = 0; k < S_PIECE; ++k)
              if ((far >> (k / SCALE_TOKENS)) & 1u)
                share += fast_exp2(fmaf(__uint_as_float(v[k]), score_factor(factor, of_block->key[h * 4 + k / SCALE_TOKENS]), -m_use));
            l2 = add2(l2, pair(share, 0.0f));
          }
          if (i > 0 || h > 0) {     // O = O * corr in tensor memory, when every product issued so far is complete
            ok = h > 0 ? wait_pv(i, 0) : wait_pv(i - 1, 1);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 16) {      // (the scores are still held)
              uint32_t t[16];
              tmem_load16_nowait(o_addr + c0, t);
              tmem_wait_loads();
#pragma unroll
              for (int k = 0; k < 16; ++k) t[k] = __float_as_uint(__uint_as_float(t[k]) * corr);
              tmem_store16(o_addr + c0, t);
            }
          }
        }
        if (!ok) break;
        tmem_wait_stores();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&p_full[g * 2 + h]);
      }
      if (!ok) break;
    }
    float l_odd;
    unpair(l2, l, l_odd);
    l += l_odd;
    if (m == INFINITY) l = __int_as_float(0x7fc00000);      // scores beyond float32
    if (ok && my_n > 0) ok = wait_pv(my_n - 1, 1) && !*abort_flag;
    if (!ok) {
      *abort_flag = 1;
      atomicCAS(a.error_word, 0, ERR_SOFTMAX);
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (n_splits == 1 && ok && my_n > 0) {
      // ---- every thread finishes its own row: O / l (less the headroom) out of tensor memory, rounded to bfloat16, 64 bytes
      // at a time.  Heads that share a key/value head lie side by side in a token's output row, as their
      // rows do in the tile.  (The loads are warp-wide, so rows without an output still take part.)
      // the sink joins the sum, taken against the same maximum (far above it the sum is infinite, the row zero)
      if (extras.sink && row_valid) l += sink_share(sink_log2(extras, head), m);
      const float inv = l == 0.0f ? 0.0f : (row_valid ? head_gate<__nv_bfloat16>(extras, q_start + token, head) : 1.0f) * P_UNIT / l;
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
    // A warp takes 128 columns at a time: a row, or two rows at head size 64.  All blocks' numbers are asked for at once (a trip to another
    // block's memory takes as long as to L2), a row's maxima and sums by one lane a block.
    constexpr int LANES = D / 4, ROWS = 32 / LANES;
    const int c4 = lane % LANES, owned = BLOCK_ROWS / n_splits;
#pragma unroll 1
    for (int i = warp * ROWS; i < owned; i += NUM_THREADS / 32 * ROWS) {
      const int row = (i + lane / LANES) * n_splits + split, packed = row0 + row;
      const bool there = i + lane / LANES < owned && packed < n_rows;
      const uint32_t local = smem_u32(states + (size_t)(there ? row : 0) * STATE);
      float4 v[MAX_SPLITS];
      const float4 ml = c4 < n_splits ? load_peer4(peer_smem(local, c4) + D * 4) : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int z = 0; z < MAX_SPLITS; ++z) v[z] = z < n_splits ? load_peer4(peer_smem(local, z) + c4 * 16) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const int tok = there ? packed / group : 0, hd = there ? kvh * group + packed % group : 0;
      const float sink = sink_log2(extras, hd);
      float M = ml.x;
#pragma unroll
      for (int by = 1; by < MAX_SPLITS; by <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, by));      // (of the first eight lanes of a row)
      M = fmaxf(__shfl_sync(0xffffffffu, M, lane & ~(LANES - 1)), sink);
      const float M_use = M == -INFINITY ? 0.0f : M;
      const float h_mine = ml.x == -INFINITY ? 1.0f : exp2f(0.5f * (ml.x - M_use));      // without a maximum: zeros, or NaN to be handed on
      const float part_mine = ml.y * h_mine * h_mine, f_mine = h_mine * h_mine;
      float L = sink_share(sink, M_use);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int z = 0; z < MAX_SPLITS; ++z) {
        const float f = __shfl_sync(0xffffffffu, f_mine, (lane & ~(LANES - 1)) + z), part = __shfl_sync(0xffffffffu, part_mine, (lane & ~(LANES - 1)) + z);
        L += part;
        acc.x += v[z].x * f, acc.y += v[z].y * f, acc.z += v[z].z * f, acc.w += v[z].w * f;
      }
      const float inv = L == 0.0f ? 0.0f : head_gate<__nv_bfloat16>(extras, q_start + tok, hd) * P_UNIT / L;
      if (there)
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
// (the largest power of two that divides the page size, up to 128), swizzled as codes_swizzled says.
extern "C" int llm_cache8_prompt_pool_map(void* map_out, const void* base, long long rows, int box_rows) {
  if ((reinterpret_cast<uintptr_t>(base) & 15) || rows <= 0 || rows > 0x7fffffffLL || box_rows < SCALE_TOKENS || BN % box_rows) return ERR_BAD_SIZE;
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return 1000 + (int)cudaErrorNotSupported;
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
  static unsigned long long raised = 0;
  const unsigned long long here = device_bit();
  if (!(raised & here)) {
    if (cudaFuncSetAttribute(cache8_prompt_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(cache8_prompt_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES) != cudaSuccess)
      return launch_status();
    raised |= here;
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
