// Softmax attention of requests that bring very few rows (tokens x query heads of one key/value head: at most 16) over a cache of
// e4m3 codes (cache8.cuh): the decode step, and steps of a few tokens.  It is to such a cache what attention_decode.cu is to a
// bfloat16 one (cuongvng/bare-cuda-4gib engine/kernels/attention_qk.cu:49-68, softmax.cu:28-42, attention_av.cu:24-44).
//
//   s[k] = scale * 2^e_K(k) * (q . K_k)     p = softmax over the visible k     out = sum_k p[k] 2^e_V(k) V_k
//
// The codes are all that is worth bandwidth (2 head_dim bytes a key against a few hundred bytes for the rest), so the kernel is built
// around their way into the tensor cores:
//  * A warp takes 16 keys at a time: one scale block, whose keys are one piece of memory and whose values are another.  It asks for STAGES such
//    blocks ahead, as TMA copies into a ring of its own (one warp's ring is nobody else's: no warp waits for another).
//  * The products are turned around: S^T = K Q^T and O^T = V^T P^T, with the codes as the left operand (16 keys or 16 channels) and up
//    to 8 query rows as the right one, which takes half the instructions of the usual way round for a group of 4 or 8 heads.  The order of the
//    inner dimension is free, so a thread takes 16 neighbouring codes a load: of a key, thread t of four takes 16 channels of every 64 and uses them
//    four at a time; of a value, the eight threads of a column take an eighth of the channels each.  Row g of the left operand is key
//    g, or g ^ 4 for odd g: then the swizzled loads of keys and values meet every bank once (values of head size 64 twice).
//  * A code becomes a half by one conversion for two; halves hold e4m3 exactly.  The scale of the keys joins the factor of
//    the scores.  A weight goes into P together with its block's value scale: P = 2^(s + e_V - m + 7) with m the running maximum of s + e_V,
//    while the sum takes P 2^(-e_V - 7); so a half of P is relative to what the row's keys can add to its output, and O needs no factor but the 2^-7 at
//    the end.  (The 2^7: weights keep a half's eleven bits down to 2^-21 of the row's largest, 15 nats below it, have an absolute step of 2^-31 of it from there on,
//    and are lost from O below 2^-32.)
//    Float32 drops a P below 2^-126, and with it a share of that times 2^(largest e_V - e_V) of the sum: nothing where e_V is of the size of the
//    others', all of it for a block of zeros (e_V = -100) beside values in the millions.  Blocks with e_V below FAR_VALUES take 2^(s - m) itself, so
//    that no share above 2^-26 is lost while the largest value is below 448 * 2^60.  (A test a block, which costs nothing here.)  For the same reason a
//    sum goes from one maximum to a larger one by way of half their distance, twice: m of a row that has seen only zeros may lie 2^200 below.
//    Queries become halves times a power of two of their row's own (exact but for entries 2^24 below the row's largest).
//  * The maximum that the exponentials are taken against moves only when a score has outgrown it by 2^8: until then 16 keys need no
//    exchange between threads but one vote.
//  * The key blocks of a request are dealt round-robin to the warps of a cluster of up to 8 thread blocks.  A block merges its
//    warps' states in shared memory and sends row r to block r % n_splits of the cluster, which merges in index order: no
//    scratch in global memory, no atomics, no second launch.
//  * Blocks of keys that lie wholly below the step's first new position are asked for before the kernel waits for the one before it.
// One B200, 32 / 8 heads of 128: 8 requests of 8,192 positions 24.0 us (5.6 TB/s, 0.86 of the copy rate; over a bfloat16 cache 44.5), 64 of 2,000
// to 8,191 115 us (5.9 TB/s).  What is left is the start of a block (its lists, then its first pages, then its first keys) and its merge.  Where a warp
// has few keys they are most of it: 64 requests of 2,047 (32 / 4 heads of 64) 17.6 us (3.9 TB/s), 32 of 1,900 11.1 (2.8; over bfloat16 12.2).
// 9 to 16 rows (NT 2) leave one block an SM: 64 requests of 8,192 with 16 heads on one of 128 49.6 us (2.7 TB/s), 8 of them 14.4 (1.2).

#include "cache8.cuh"

#include <cuda.h>
#include <cuda_fp16.h>
#include <string.h>

#ifndef HEAD_DIM
#define HEAD_DIM 64
#endif

namespace {

constexpr int D = HEAD_DIM;
static_assert(D == 64 || D == 128, "HEAD_DIM must be 64 or 128");
constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int UNIT = SCALE_TOKENS;             // keys a warp takes at a time
constexpr int KG = D / 64;                     // 64-channel groups of a key
constexpr int TILES = D / 16;                  // 16-channel tiles of the output
constexpr int VW = D / 32;                     // 32-bit words of a value that a thread takes (an eighth of its channels)
constexpr int FEW_ROWS = 16;
constexpr float RESCALE_STEP = 8.0f;           // base-2 units
constexpr int HEADROOM = 7;                    // with the step above, what a half can hold over one: 2^15
constexpr float P_UNIT = 1.0f / (1 << HEADROOM);
static_assert(HEADROOM <= 126 - SCALE_MOST, "the sum takes 2^(-e_V - HEADROOM)");
constexpr int FAR_VALUES = -40;
constexpr float MOST_FACTOR = 3.40282347e38f;
constexpr int UNIT_BYTES = UNIT * D;           // keys, or values, of one scale block
constexpr int STAGES = D == 128 ? 3 : 6;       // scale blocks a warp has in flight: 96 KB a thread block, two of which share an SM
constexpr int RING_BYTES = WARPS * STAGES * 2 * UNIT_BYTES;
constexpr unsigned long long WAIT_LIMIT_NS = 1000000000ull;
constexpr int ERR_DECODE = 46, ERR_DECODE_LAYOUT = 47;
constexpr int STATE = D + 4;                   // floats of a row's state: D sums, the maximum, the sum

struct DecodeArgs {
  const __nv_bfloat16* q;      // [rows][q_heads * D]
  __nv_bfloat16* out;
  Cache8 cache;
  long long page_rows, k_row0, v_row0;   // the pool seen as rows of D codes
  StepLists lists;
  int q_heads;
  float scale_log2;
  int window;
  int ordered;                 // longest requests first
  AttentionExtras extras;
  int* error_word;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t peer_smem(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two e4m3 codes (the lower half of `lo`, the upper half for the second) as two halves.
__device__ __forceinline__ void halves(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {   // an 8 x 8 matrix of halves spread over the warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ unsigned long long global_timer() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
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
// Waits for a copy; false after about a second, with the error word set.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, int* error_word) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long start = global_timer();
  for (unsigned spins = 0;; ++spins) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((spins & 63u) == 63u && global_timer() - start > WAIT_LIMIT_NS) {
      atomicCAS(error_word, 0, ERR_DECODE);
      return false;
    }
  }
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
}
// Byte offset of chunk `chunk` (16 codes) of row `row` in a block as TMA writes it: 128-byte swizzle for rows of 128 bytes, 64-byte swizzle
// for rows of 64.
__device__ __forceinline__ uint32_t codes_swizzled(int row, int chunk) {
  return (uint32_t)(row * D + ((D == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3)) << 4));
}
// Which of 16 keys is row (or inner index) i of the products.
__device__ __forceinline__ int key_of(int i) { return (i & 1) ? i ^ 4 : i; }

__device__ __forceinline__ void load_shared4(uint32_t* w, uint32_t at) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_shared2(uint32_t* w, uint32_t at) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
}

// NT: groups of 8 query rows.  EXTRAS: whether blocks of positions, a sink or a gate may be asked for.
template <int NT, bool EXTRAS>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 2 : 1) cache8_decode_kernel(const __grid_constant__ CUtensorMap pool_map, const DecodeArgs a) {
  constexpr int ROWS = 8 * NT;
  const AttentionExtras extras = EXTRAS ? a.extras : AttentionExtras{0, nullptr, nullptr, 0};
  extern __shared__ __align__(1024) uint8_t ring[];         // [WARPS][STAGES][keys, values][UNIT_BYTES]
  const int n_splits = gridDim.z, split = blockIdx.z, owned_rows = (ROWS + n_splits - 1) / n_splits;
  float* st = reinterpret_cast<float*>(ring);             // [WARPS][ROWS][STATE]: this block's warps, when they are done with the ring
  float* recv = reinterpret_cast<float*>(ring + RING_BYTES);   // [n_splits][owned_rows][STATE]: written by the cluster
  uint64_t* full = reinterpret_cast<uint64_t*>(recv + n_splits * owned_rows * STATE);   // [WARPS][STAGES]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[warp * STAGES + i], 1);      // (its own warp's alone)
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&pool_map)) : "memory");
  }
  __syncwarp();
  const int seq = a.ordered ? a.lists.order[blockIdx.x] : blockIdx.x;
  const int part = blockIdx.y / a.cache.kv_heads, kvh = blockIdx.y - part * a.cache.kv_heads, row0 = part * ROWS;   // row0: of the request's rows, this block's first
  const int group = a.q_heads / a.cache.kv_heads;
  const int q_start = a.lists.seq_q_start[seq], q_len = a.lists.seq_q_len[seq], kv_len = a.lists.seq_kv_len[seq], n_rows = q_len * group;
  if (n_rows <= row0 || n_rows > FEW_ROWS) {              // nothing, or the prompt kernel's: the same for the whole cluster
    if (blockIdx.x + blockIdx.y == 0) pdl_wait();      // (a kernel may not end ahead of those before it; the other blocks hold up none that has work)
    return;
  }
  if (smem_u32(ring) & 1023) {      // never seen; the swizzled blocks need it
    if (threadIdx.x == 0) atomicCAS(a.error_word, 0, ERR_DECODE_LAYOUT);
    pdl_wait();
    return;
  }
  if (n_splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this block runs: its memory may be written
  const int pos0 = kv_len - q_len;
  const int lo_key = first_visible_key(pos0, a.window, extras.chunk);
  const int max_lo = first_visible_key(kv_len - 1, a.window, extras.chunk);   // from here on no row's bound hides a key
  const int u_lo = lo_key / UNIT, u_hi = (kv_len - 1) / UNIT;
  const int stride = WARPS * n_splits, first = u_lo + split * WARPS + warp;
  const int n_units = first > u_hi ? 0 : (u_hi - first) / stride + 1;         // this warp's: first, first + stride, ...
  const int closed = pos0 / UNIT;                                             // units from here on this step's append may write

  // Where the warp's units lie, looked up 32 at a time and 32 ahead: lane i knows unit i of the stretch at hand and of the next.
  struct Places {
    int row;                 // of the pool, without the cache's own offset, or -1
    float k_scale;
    int v_exponent;
  };
  auto look_up = [&](int from) {
    Places p{-1, 0.0f, 0};
    if (from + lane < n_units) {
      const int unit = first + (from + lane) * stride, page = page_of(a.cache, seq, unit * UNIT);
      if (page >= 0) {
        const int in_page = unit * UNIT % a.cache.page_tokens;
        p.row = (int)((long long)page * a.page_rows + (long long)kvh * a.cache.page_tokens + in_page);
        const long long at = (long long)page * a.cache.scale_stride + (long long)kvh * (a.cache.page_tokens / UNIT) + in_page / UNIT;
        p.k_scale = __ldcg(a.cache.k_scale + at);
        p.v_exponent = max(exponent_of(__ldcg(a.cache.v_scale + at)), SCALE_LEAST);      // (a scale that nothing has written is zero)
      }
    }
    return p;
  };
  Places here{-1, 0.0f, 0}, ahead{-1, 0.0f, 0};
  const uint32_t my_ring = smem_u32(ring) + warp * STAGES * 2 * UNIT_BYTES;
  uint64_t* my_full = full + warp * STAGES;
  // asks for unit j, whose row the caller knows, into its stage (a unit without a page: nothing comes, and nothing is waited for long)
  auto request = [&](int j, int row) {
    if (lane == 0) {
      const uint32_t to = my_ring + (j % STAGES) * 2 * UNIT_BYTES;
      mbar_expect_tx(&my_full[j % STAGES], row >= 0 ? 2 * UNIT_BYTES : 0);
      if (row >= 0) {
        tma_load_2d(to, &pool_map, &my_full[j % STAGES], 0, (int)(row + a.k_row0));
        tma_load_2d(to + UNIT_BYTES, &pool_map, &my_full[j % STAGES], 0, (int)(row + a.v_row0));
      }
    }
  };
  bool waited = false;
  if (n_units > 0) {
    // the append ahead of this kernel may still write the open blocks, codes and scales: only stretches below them may be read ahead
    // of the wait
    if (first + (min(n_units, 32) - 1) * stride >= closed) pdl_wait(), waited = true;
    here = look_up(0);
#pragma unroll
    for (int j = 0; j < STAGES; ++j) {
      const int row = __shfl_sync(0xffffffffu, here.row, j);
      if (j < n_units) request(j, row);
    }
  }
  if (!waited) pdl_wait();
  ahead = look_up(32);

  // ---- the query rows as halves, times a power of two that brings a row's largest entry to [2^10, 2^11)
  uint32_t qf[NT][KG * 4][2];
  float factor[NT][2];       // of rows 2 t and 2 t + 1: scale * log2(e) times that power back
  int row_pos[NT][2], row_lo[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int R = row0 + n * 8 + g;
    uint4 raw[KG][2];
#pragma unroll
    for (int i = 0; i < KG; ++i) raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
    if (R < n_rows) {
      const __nv_bfloat16* src = a.q + ((long long)(q_start + R / group) * a.q_heads + kvh * group + R % group) * D + 16 * t;
#pragma unroll
      for (int i = 0; i < KG; ++i) {
        raw[i][0] = *reinterpret_cast<const uint4*>(src + i * 64);
        raw[i][1] = *reinterpret_cast<const uint4*>(src + i * 64 + 8);
      }
    }
    float most = 0.0f;
    const __nv_bfloat162* pairs = reinterpret_cast<const __nv_bfloat162*>(raw);
#pragma unroll
    for (int i = 0; i < KG * 8; ++i) most = fmaxf(most, fmaxf(fabsf(__low2float(pairs[i])), fabsf(__high2float(pairs[i]))));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = most > 0.0f ? min(max(exponent_of(most) - 10, -100), 116) : 0;
    const float down = most < INFINITY ? power_of_two(-e) : __int_as_float(0x7fc00000);      // (an infinite entry makes the row NaN, as in the prompt kernel)
#pragma unroll
    for (int i = 0; i < KG * 8; ++i)
      qf[n][i >> 1][i & 1] = pack_half(__low2float(pairs[i]) * down, __high2float(pairs[i]) * down);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int col = 2 * t + h, C = row0 + n * 8 + col;
      factor[n][h] = a.scale_log2 * power_of_two(__shfl_sync(0xffffffffu, e, col * 4));
      row_pos[n][h] = C < n_rows ? pos0 + C / group : -1;
      row_lo[n][h] = first_visible_key(row_pos[n][h], a.window, extras.chunk);
    }
  }

  float m[NT][2], l[NT][2], o[NT][TILES][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < TILES; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
  }

  for (int j = 0; j < n_units; ++j) {
    if (j > 0 && (j & 31) == 0) here = ahead, ahead = look_up(j + 32);
    const int row = __shfl_sync(0xffffffffu, here.row, j & 31);
    const float ks = __shfl_sync(0xffffffffu, here.k_scale, j & 31);
    const int ev = __shfl_sync(0xffffffffu, here.v_exponent, j & 31);
    const int later = j + STAGES;                          // the unit that takes this one's stage
    const int later_row = (later ^ j) & 32 ? __shfl_sync(0xffffffffu, ahead.row, later & 31) : __shfl_sync(0xffffffffu, here.row, later & 31);
    const bool landed = mbar_wait(&my_full[j % STAGES], (uint32_t)(j / STAGES) & 1u, a.error_word);
    if (row < 0) {                  // a page that a window has given back: no row sees it
      __syncwarp();                 // (every lane has seen this phase)
      if (later < n_units) request(later, later_row);
      continue;
    }
    const uint32_t k_at = my_ring + (j % STAGES) * 2 * UNIT_BYTES, v_at = k_at + UNIT_BYTES;
    uint32_t kc[2][KG][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < KG; ++i) load_shared4(kc[h][i], k_at + codes_swizzled(key_of(g) + 8 * h, i * 4 + t));
    const int key0 = (first + j * stride) * UNIT;
    float s[NT][4], s_odd[NT][4];      // two chains of products instead of one
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = s_odd[n][e] = 0.0f;
#pragma unroll
    for (int i = 0; i < KG; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t a0, a1, a2, a3;
        halves(kc[0][i][w], a0, a2);
        halves(kc[1][i][w], a1, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(w & 1 ? s_odd[n] : s[n], a0, a1, a2, a3, qf[n][i * 4 + w][0], qf[n][i * 4 + w][1]);
      }
    const bool all_visible = key0 + UNIT - 1 <= pos0 && key0 >= max_lo;
    float c[NT][2];       // infinite times a score of zero would be no number (a NaN of the keys' scale stays one)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) c[n][h] = factor[n][h] * ks, c[n][h] = c[n][h] > MOST_FACTOR ? MOST_FACTOR : c[n][h];
    bool grown = !landed;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int h = e & 1;
        float v = fmaf(s[n][e] + s_odd[n][e], c[n][h], (float)ev);
        if (!all_visible) {
          const int key = key0 + key_of(g) + 8 * (e >> 1);
          if (key > row_pos[n][h] || key < row_lo[n][h]) v = -INFINITY;
        }
        s[n][e] = v;
        grown |= v > m[n][h] + RESCALE_STEP;
      }
    if (__any_sync(0xffffffffu, grown)) {
      if (!__all_sync(0xffffffffu, landed)) {      // the copies on their way land before the warp goes to its barriers and its end
        for (int i = j; i < min(j + STAGES, n_units); ++i) mbar_wait(&my_full[i % STAGES], (uint32_t)(i / STAGES) & 1u, a.error_word);
        break;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = fmaxf(s[n][h], s[n][h + 2]);
#pragma unroll
          for (int by = 4; by < 32; by <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, by));
          const float m_new = fmaxf(m[n][h], top);
          const float down = m_new == -INFINITY ? 0.0f : m[n][h] - m_new, half_way = fast_exp2(0.5f * down), corr = fast_exp2(down);
          m[n][h] = m_new;
          l[n][h] = l[n][h] * half_way * half_way;
#pragma unroll
          for (int i = 0; i < TILES; ++i) o[n][i][h] *= corr, o[n][i][h + 2] *= corr;
        }
    }
    uint32_t pf[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float m0 = m[n][0] == -INFINITY ? 0.0f : m[n][0] - HEADROOM, m1 = m[n][1] == -INFINITY ? 0.0f : m[n][1] - HEADROOM;
      const float p0 = fast_exp2(s[n][0] - m0), p1 = fast_exp2(s[n][1] - m1), p2 = fast_exp2(s[n][2] - m0), p3 = fast_exp2(s[n][3] - m1);
      if (ev >= FAR_VALUES) {       // the same for the whole warp
        l[n][0] = fmaf(p0 + p2, power_of_two(-ev - HEADROOM), l[n][0]);
        l[n][1] = fmaf(p1 + p3, power_of_two(-ev - HEADROOM), l[n][1]);
      } else {
        const float e = (float)(ev + HEADROOM);
        l[n][0] += fast_exp2(s[n][0] - e - m0) + fast_exp2(s[n][2] - e - m0);
        l[n][1] += fast_exp2(s[n][1] - e - m1) + fast_exp2(s[n][3] - e - m1);
      }
      pf[n][0] = transposed(pack_half(p0, p1));
      pf[n][1] = transposed(pack_half(p2, p3));
    }
    uint32_t vc[4][VW];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = key_of(2 * t + (i & 1)) + 8 * (i >> 1);
      if (D == 128) load_shared4(vc[i], v_at + codes_swizzled(key, g));
      else load_shared2(vc[i], v_at + codes_swizzled(key, g >> 1) + (g & 1) * 8);
    }
    if (key0 + UNIT > kv_len) {     // behind the last key a page may hold anything, and zero times NaN is not zero
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key0 + key_of(2 * t + (i & 1)) + 8 * (i >> 1) >= kv_len)
#pragma unroll
          for (int w = 0; w < VW; ++w) vc[i][w] = 0;
    }
#pragma unroll
    for (int w = 0; w < VW; ++w)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // channels 4 w + 2 half and + 1 of this thread's eighth, of its four keys
        const uint32_t pick = half ? 0x7362u : 0x5140u;
        uint32_t a0, a1, a2, a3;
        halves(__byte_perm(vc[0][w], vc[1][w], pick), a0, a1);
        halves(__byte_perm(vc[2][w], vc[3][w], pick), a2, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * w + half], a0, a1, a2, a3, pf[n][0], pf[n][1]);
      }
    // behind the products: what every lane read of the stage has arrived in its registers (a load that is merely on its way when the
    // copy is asked for may be overtaken by it)
    __syncwarp();
    if (later < n_units) request(later, later_row);
  }

  __syncthreads();      // every warp is done with its ring
  // ---- the warps' states into shared memory: row C of the tile, channels g * D / 8 + 2 i (+ 1)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float sum = l[n][h];
#pragma unroll
      for (int by = 4; by < 32; by <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, by);
      float* row = st + ((size_t)warp * ROWS + n * 8 + 2 * t + h) * STATE;
#pragma unroll
      for (int i = 0; i < TILES; i += 2)
        *reinterpret_cast<float4*>(row + g * (D / 8) + 2 * i) = make_float4(o[n][i][h], o[n][i][h + 2], o[n][i + 1][h], o[n][i + 1][h + 2]);
      if (g == 0) row[D] = m[n][h], row[D + 1] = sum;
    }
  __syncthreads();
  if (n_splits > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // all blocks of the cluster have started
  // ---- the block's warps merged, four channels a thread; row r goes to block r % n_splits
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += THREADS) {
    const int r = i / (D / 4), c4 = i % (D / 4);
    if (row0 + r >= n_rows) continue;
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, st[((size_t)w * ROWS + r) * STATE + D]);
    const float M_use = M == -INFINITY ? 0.0f : M;        // (a row of NaN has no maximum, but sums)
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float* from = st + ((size_t)w * ROWS + r) * STATE;
      const float half_way = from[D] == -INFINITY ? 1.0f : exp2f(0.5f * (from[D] - M_use)), f = half_way * half_way;   // without a maximum: zeros, or NaN to be handed on
      const float4 v = *reinterpret_cast<const float4*>(from + c4 * 4);
      L += from[D + 1] * half_way * half_way;
      acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
    }
    const uint32_t local = smem_u32(recv + ((size_t)split * owned_rows + r / n_splits) * STATE);
    const uint32_t dst = n_splits > 1 ? peer_smem(local, r % n_splits) : local;
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + c4 * 16), "f"(acc.x), "f"(acc.y), "f"(acc.z), "f"(acc.w) : "memory");
    if (c4 == 0) asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst + D * 4), "f"(M), "f"(L) : "memory");
  }
  if (n_splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();

  // ---- the rows this block owns, merged over the blocks in index order
  for (int i = threadIdx.x; i < owned_rows * (D / 4); i += THREADS) {
    const int slot = i / (D / 4), c4 = i % (D / 4), r = slot * n_splits + split;
    if (row0 + r >= n_rows) continue;
    const int token = (row0 + r) / group, head = kvh * group + (row0 + r) % group;
    const float sink = sink_log2(extras, head);            // joins the row's sum here, once
    float M = sink;
#pragma unroll 8
    for (int z = 0; z < n_splits; ++z) M = fmaxf(M, recv[((size_t)z * owned_rows + slot) * STATE + D]);
    const float M_use = M == -INFINITY ? 0.0f : M;
    float L = sink_share(sink, M_use);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int z = 0; z < n_splits; ++z) {
      const float* from = recv + ((size_t)z * owned_rows + slot) * STATE;
      const float half_way = from[D] == -INFINITY ? 1.0f : exp2f(0.5f * (from[D] - M_use)), f = half_way * half_way;
      const float4 v = *reinterpret_cast<const float4*>(from + c4 * 4);
      L += from[D + 1] * half_way * half_way;
      acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
    }
    const float inv = L == 0.0f ? 0.0f : head_gate<__nv_bfloat16>(extras, q_start + token, head) * P_UNIT / L;
    *reinterpret_cast<uint2*>(a.out + ((long long)(q_start + token) * a.q_heads + head) * D + c4 * 4) =
        make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
}

static_assert(WARPS * FEW_ROWS * STATE * 4 <= RING_BYTES, "the warps' states lie over the ring");
size_t smem_bytes(int rows, int n_splits) {
  return RING_BYTES + (size_t)n_splits * ((rows + n_splits - 1) / n_splits) * STATE * 4 + WARPS * STAGES * 8;
}

template <int NT>
int launch(const CUtensorMap& map, const DecodeArgs& a, int parts, int n_splits, cudaStream_t stream) {
  static unsigned long long raised = 0;
  const unsigned long long here = device_bit();
  if (!(raised & here)) {
    const int most = (int)(RING_BYTES + (8 * NT + 8) * STATE * 4 + WARPS * STAGES * 8);
    if (cudaFuncSetAttribute(cache8_decode_kernel<NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess ||
        cudaFuncSetAttribute(cache8_decode_kernel<NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
      return launch_status();
    raised |= here;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.lists.n_seqs, a.cache.kv_heads * parts, n_splits);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem_bytes(8 * NT, n_splits);
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
  const AttentionExtras& x = a.extras;
  cudaLaunchKernelEx(&cfg, x.chunk > 0 || x.sink || x.gate ? cache8_decode_kernel<NT, true> : cache8_decode_kernel<NT, false>, map, a);
  return launch_status();
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

// Writes the 128-byte tensor map of a pool of `rows` rows of D codes starting at `base` (16-byte aligned), boxes of one scale block, swizzled as
// codes_swizzled says.
extern "C" int llm_cache8_decode_pool_map(void* map_out, const void* base, long long rows) {
  if ((reinterpret_cast<uintptr_t>(base) & 15) || rows <= 0 || rows > 0x7fffffffLL) return ERR_BAD_SIZE;
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return 1000 + (int)cudaErrorNotSupported;
  cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)D};
  cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)UNIT};
  cuuint32_t elem[2] = {1, 1};
  CUresult r = fn(reinterpret_cast<CUtensorMap*>(map_out), CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 2000 + (int)r;
}

// Every request with 1 .. 16 packed rows (q_len * q_heads / kv_heads); the others' blocks return at once.  `rows`: the most packed rows
// that such a request of the step brings.  More than 8 take the kernel for 16, or (`parts` 2) two blocks of the kernel for 8, of which
// the second one of a request with no more than 8 returns at once.  n_splits (1, 2, 4 or 8) blocks share a
// request's keys.  `ordered`: the longest requests' blocks start first
// (worth its look-up where not all blocks run at once).  `pool_map`: llm_cache8_decode_pool_map over `pool_base`, in which the cache's codes lie.  chunk, sink, gate and gate_stride: `AttentionExtras`; 0 and null: none.
extern "C" int llm_cache8_attention_decode(const void* q, void* out, const Cache8* cache, const void* pool_map, const void* pool_base,
                                           const StepLists* lists, int n_splits, int ordered, int rows, int parts, int q_heads, float scale, int window, int chunk,
                                           const float* sink, const void* gate, long long gate_stride, int* error_word,
                                           cudaStream_t stream) {
  if (lists->n_seqs <= 0) return 0;
  const Cache8& c = *cache;
  if (c.head_dim != D || c.kv_heads <= 0 || q_heads <= 0 || q_heads % c.kv_heads || c.kv_heads > 32767 || (parts != 1 && parts != 2) || c.page_tokens <= 0 ||
      c.page_tokens % SCALE_TOKENS || (n_splits != 1 && n_splits != 2 && n_splits != 4 && n_splits != 8) || rows < 1 || rows > FEW_ROWS)
    return ERR_BAD_SIZE;
  const uintptr_t all = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(c.k) |
                        reinterpret_cast<uintptr_t>(c.v) | (uintptr_t)c.page_stride;
  const long long k_off = reinterpret_cast<const char*>(c.k) - reinterpret_cast<const char*>(pool_base);
  const long long v_off = reinterpret_cast<const char*>(c.v) - reinterpret_cast<const char*>(pool_base);
  if ((all & 15) || k_off < 0 || v_off < 0 || k_off % D || v_off % D || c.page_stride % D) return ERR_BAD_ALIGN;
  DecodeArgs a{reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<__nv_bfloat16*>(out), c, c.page_stride / D, k_off / D,
               v_off / D, *lists, q_heads, scale * 1.4426950408889634f, window, ordered, AttentionExtras{chunk, sink, gate, gate_stride}, error_word};
  CUtensorMap map;   // the caller's buffer need not be 64-byte aligned
  memcpy(&map, pool_map, sizeof(CUtensorMap));
  return rows <= 8 || parts == 2 ? launch<1>(map, a, parts, n_splits, stream) : launch<2>(map, a, 1, n_splits, stream);
}
