// The append to a cache of e4m3 codes: a step's projections [q | k | v] -> q turned by position (bfloat16), k turned by position
// and v written as codes with a power-of-two scale per 16 positions, key/value head and keys or values (cache8.cuh).  It is to
// such a cache what rope_cache_write is to a bfloat16 one (cuongvng/bare-cuda-4gib engine/kernels/rope.cu:18-55,
// kv_cache_write.cu:10-33).
//
//   (x_p, x_p+half) -> (x_p cos - x_p+half sin, x_p+half cos + x_p sin), angle = position * inv_freq[p]
//   a = the largest entry of the block's new tokens in size; e = the smallest with a <= 448 * 2^e
//   block opened by an earlier step with scale 2^f: e = max(e, f), and if e > f its codes become round(code * 2^(f - e))
//   code = round(x * 2^-e), to nearest, ties to even
//
// One thread block per (written block of 16 positions, key/value head): it holds the head's new keys and values of those
// positions in registers (a thread 16 entries of each of one token), so they are read once, and it alone
// settles the two scales: no atomics, no second pass.  The query heads that share the key/value head go through the same block:
// their angles are the ones the keys need, computed once into shared memory; their first two rows are asked for together with the keys.
// Bound by memory for prompts (projections in, queries out), by its trips to memory for decoding steps.  One B200, in a graph: 8 decoding
// requests (32 / 8 heads of 128) 2.4 us, 64 with three partial results (32 / 4 heads of 64) 3.3, a prompt's 2,048 tokens (32 / 8 heads of 128)
// 8.3 (5.6 TB/s, most of it from L2), 32,768 tokens 136 (5.4 TB/s).

#include "cache8.cuh"

#include <cuda_fp8.h>

namespace {

constexpr int TOKENS = SCALE_TOKENS;

struct AppendArgs {
  const void* qkv;             // [partials][rows][(q_heads + 2 kv_heads) * head_dim]
  int n_partials;
  long long partial_stride;
  __nv_bfloat16* q_out;        // [rows][q_heads * head_dim]
  Cache8 cache;
  StepLists lists;
  const float* inv_freq;       // null: no rotation
  int q_heads, write_cache;
};

// Eight neighbouring entries.
__device__ __forceinline__ void load8(float (&x)[8], const float* p) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(float (&x)[8], const __nv_bfloat16* p) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
// N times eight entries of the sum of the partial results (ONE: there is one), a partial result's all on their way at once.
template <typename T, bool ONE, int N>
__device__ __forceinline__ void load_sums(float (&x)[N][8], const T* const (&p)[N], int n_partials, long long stride) {
#pragma unroll
  for (int k = 0; k < N; ++k) load8(x[k], p[k]);
  if (ONE) return;
  for (int i = 1; i < n_partials; ++i) {
    float y[N][8];
#pragma unroll
    for (int k = 0; k < N; ++k) load8(y[k], p[k] + i * stride);
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] += y[k][e];
  }
}

// A query's two pieces on their way: as they were loaded where that is all there is to them, which takes half the registers.
template <typename T, bool ONE>
struct Pieces {
  float x[2][8];
  __device__ __forceinline__ void load(const T* lo, const T* hi, int n_partials, long long stride) {
    const T* const p[2] = {lo, hi};
    load_sums<T, ONE>(x, p, n_partials, stride);
  }
  __device__ __forceinline__ void get(float (&lo)[8], float (&hi)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = x[0][i], hi[i] = x[1][i];
  }
};
template <>
struct Pieces<__nv_bfloat16, true> {
  uint4 raw[2];
  __device__ __forceinline__ void load(const __nv_bfloat16* lo, const __nv_bfloat16* hi, int, long long) {
    raw[0] = *reinterpret_cast<const uint4*>(lo), raw[1] = *reinterpret_cast<const uint4*>(hi);
  }
  __device__ __forceinline__ void get(float (&lo)[8], float (&hi)[8]) const {
    load8(lo, reinterpret_cast<const __nv_bfloat16*>(&raw[0])), load8(hi, reinterpret_cast<const __nv_bfloat16*>(&raw[1]));
  }
};

// (lo, hi) turned by the angles of `cs`: two (cos, sin) at a time, STEP apart.
template <int STEP>
__device__ __forceinline__ void turn(float (&lo)[8], float (&hi)[8], const float4* cs) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float4 t = cs[i / 2 * STEP];
    const float a = lo[i], b = hi[i], c = lo[i + 1], d = hi[i + 1];
    lo[i] = a * t.x - b * t.y;
    hi[i] = b * t.x + a * t.y;
    lo[i + 1] = c * t.z - d * t.w;
    hi[i + 1] = d * t.z + c * t.w;
  }
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The largest finite entry in size; `spoilt` if one is not finite, which then counts as zero.
__device__ __forceinline__ float largest_of(float (&x)[8], bool& spoilt) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!finite(x[i])) spoilt = true, x[i] = 0.0f;
    m = fmaxf(m, fabsf(x[i]));
  }
  return m;
}

// The smallest e with a <= 448 * 2^e = 1.75 * 2^(e + 8), within the bounds.
__device__ __forceinline__ int scale_exponent(float a) {
  const int bits = __float_as_int(a);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return min(max(e, SCALE_LEAST), SCALE_MOST);      // zero and numbers below the normal range: the least
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float f) {
  return make_uint2(codes4(x[0] * f, x[1] * f, x[2] * f, x[3] * f), codes4(x[4] * f, x[5] * f, x[6] * f, x[7] * f));
}
// Four codes times `factor`, rounded anew.
__device__ __forceinline__ uint32_t rescaled(uint32_t codes, float factor) {
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffff), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E4M3);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  return codes4(x.x * factor, x.y * factor, y.x * factor, y.y * factor);
}
__device__ __forceinline__ void rescale16(uint8_t* at, float factor) {
  uint4* p = reinterpret_cast<uint4*>(at);
  const uint4 old = *p;
  *p = make_uint4(rescaled(old.x, factor), rescaled(old.y, factor), rescaled(old.z, factor), rescaled(old.w, factor));
}
__device__ __forceinline__ uint4 bf16x8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 896 threads an SM where there is one result to read (768: 2,048 tokens of 32 / 8 heads of 128 in 11.8 us where this took 9.2; 1,024: 9.7,
// registers spilled; a single float32 result spills 76 to 80 bytes already), 512 with partial ones, whose loads on their way take more (2,048 tokens with four results 33.3 us; 768 threads 34.0; a
// piece's results one after another 54).
template <int D, typename T, bool ONE>
__global__ void __launch_bounds__(TOKENS * (D / 16), (D == 128 ? 1 : 2) * (ONE ? 7 : 4)) cache8_append_kernel(const AppendArgs a) {
  constexpr int CHUNKS = D / 16, HALF = D / 2, THREADS = TOKENS * CHUNKS, AHEAD = ONE ? 2 : 1;
  pdl_launch_dependents();
  // (cos, sin) of pairs 8 c + 2 k and 8 c + 2 k + 1 at [token][k][c], so that the threads of a token, and at head size 64 those of two, read side
  // by side (pair after pair they would read a line in four turns: 8,192 tokens of 32 / 8 heads of 128 37.6 us, so 34.2; 32 / 4 heads of 64 15.8, 11.8)
  constexpr int ROW = 4 * CHUNKS + (D == 64 ? 4 : 0);
  __shared__ float4 angles[TOKENS][ROW];
  __shared__ float largest[2][THREADS / 32];
  const int tid = threadIdx.x, group_of = tid / CHUNKS, c = tid % CHUNKS, kvh = blockIdx.y;
  const int seq = a.lists.write_seq[blockIdx.x];
  if (seq < 0) {
    pdl_wait();
    return;
  }
  const int first = a.lists.write_block[blockIdx.x] * TOKENS;
  const int q_start = a.lists.seq_q_start[seq], kv_len = a.lists.seq_kv_len[seq], cached = kv_len - a.lists.seq_q_len[seq];
  const int lo = max(first, cached), n_new = min(first + TOKENS, kv_len) - lo;      // the block's new positions: lo ..
  const long long row0 = (long long)q_start + lo - cached;                            // their first row
  if (n_new <= 0) {        // (rows that the step does not have)
    pdl_wait();
    return;
  }
  const int page = page_of(a.cache, seq, first);
  const bool write = a.write_cache && page >= 0;
  const int in_page = first % a.cache.page_tokens;
  const long long at = (long long)page * a.cache.page_stride + ((long long)kvh * a.cache.page_tokens + in_page) * D;
  const long long scale_at = (long long)page * a.cache.scale_stride + (long long)kvh * (a.cache.page_tokens / TOKENS) + in_page / TOKENS;
  if (a.inv_freq) {
    // The angle's product in two parts, p f = hi + lo exactly: far positions keep their angle.  lo is at most half a step of hi, 1/2 at 2^24, to which
    // positions are float32 numbers; its sine and cosine by their series, off by 1.6e-6 there and by 1e-8 up to 2^22.
    for (int i = tid; i < n_new * HALF; i += THREADS) {
      const float p = (float)(lo + i / HALF), f = a.inv_freq[i % HALF], hi = p * f, rest = fmaf(p, f, -hi);
      const float r2 = rest * rest, rs = rest * fmaf(r2, fmaf(r2, 1.0f / 120, -1.0f / 6), 1.0f),
                  rc = fmaf(r2, fmaf(r2, fmaf(r2, -1.0f / 720, 1.0f / 24), -0.5f), 1.0f);
      float s, co;
      sincosf(hi, &s, &co);
      const int pair = i % HALF;
      reinterpret_cast<float2*>(&angles[i / HALF][pair % 8 / 2 * CHUNKS + pair / 8])[pair & 1] = make_float2(co * rc - s * rs, s * rc + co * rs);
    }
  }
  __syncthreads();
  pdl_wait();

  const int group = a.q_heads / a.cache.kv_heads, n_heads = a.q_heads + 2 * a.cache.kv_heads;
  const T* qkv = reinterpret_cast<const T*>(a.qkv) + row0 * n_heads * D;
  // ---- keys and values: token `group_of` of the new ones; pairs 8 c .. 8 c + 7 of the key, entries 16 c .. 16 c + 15 of the value
  const bool mine = write && group_of < n_new;
  float kv[4][8] = {};      // the key's two pieces, the value's
  float (&k_lo)[8] = kv[0], (&k_hi)[8] = kv[1], (&v_lo)[8] = kv[2], (&v_hi)[8] = kv[3];
  if (mine) {
    const T* k = qkv + ((long long)group_of * n_heads + a.q_heads + kvh) * D;
    const T* v = k + (long long)a.cache.kv_heads * D;
    const T* const pieces[4] = {k + 8 * c, k + HALF + 8 * c, v + 16 * c, v + 16 * c + 8};
    load_sums<T, ONE>(kv, pieces, a.n_partials, a.partial_stride);
  }
  // the query heads of this key/value head: (head, token) pairs dealt to the groups of threads, tokens fastest, so that
  // a block with a single new token (a decoding request) turns up to 16 heads at once
  const int n_units = n_new * group;
  Pieces<T, ONE> q_pieces[AHEAD];
  auto load_queries = [&](int from) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int u = from + i * TOKENS;
      if (u >= n_units) break;
      const T* q = qkv + ((long long)(u % n_new) * n_heads + kvh * group + u / n_new) * D;
      q_pieces[i].load(q + 8 * c, q + HALF + 8 * c, a.n_partials, a.partial_stride);
    }
  };
  auto store_queries = [&](int from) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int u = from + i * TOKENS;
      if (u >= n_units) break;
      const int token = u % n_new, head = kvh * group + u / n_new;
      float lo[8], hi[8];
      q_pieces[i].get(lo, hi);
      if (a.inv_freq) turn<CHUNKS>(lo, hi, &angles[token][c]);
      __nv_bfloat16* out = a.q_out + ((row0 + token) * a.q_heads + head) * D;
      *reinterpret_cast<uint4*>(out + 8 * c) = bf16x8(lo);
      *reinterpret_cast<uint4*>(out + HALF + 8 * c) = bf16x8(hi);
    }
  };
  load_queries(group_of);
  if (write) {        // the same for every thread of the block
    bool spoilt = false;
    if (mine && a.inv_freq) turn<CHUNKS>(k_lo, k_hi, &angles[group_of][c]);
    float k_most = fmaxf(largest_of(k_lo, spoilt), largest_of(k_hi, spoilt)), v_most = fmaxf(largest_of(v_lo, spoilt), largest_of(v_hi, spoilt));
    k_most = warp_max(k_most), v_most = warp_max(v_most);
    if ((tid & 31) == 0) largest[0][tid >> 5] = k_most, largest[1][tid >> 5] = v_most;
    spoilt = __syncthreads_or(spoilt);
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) k_most = fmaxf(k_most, largest[0][w]), v_most = fmaxf(v_most, largest[1][w]);
    int ek = scale_exponent(k_most), ev = scale_exponent(v_most);
    const int held = lo - first;                        // positions that earlier steps filled
    uint8_t *k_codes = a.cache.k + at, *v_codes = a.cache.v + at;
    if (held > 0) {
      const float k_before = a.cache.k_scale[scale_at], v_before = a.cache.v_scale[scale_at];
      const bool k_lost = isnan(k_before);
      spoilt |= k_lost;
      const int fk = k_lost ? ek : exponent_of(k_before), fv = exponent_of(v_before);
      __syncthreads();                                  // every thread has read the scales before one writes them
      ek = max(ek, fk), ev = max(ev, fv);
      if (group_of < held) {                            // the codes of those positions, should a scale have grown
        if (ek > fk) rescale16(k_codes + group_of * D + 16 * c, power_of_two(max(fk - ek, -126)));
        if (ev > fv) rescale16(v_codes + group_of * D + 16 * c, power_of_two(max(fv - ev, -126)));
      }
    }
    if (tid == 0) {
      a.cache.k_scale[scale_at] = spoilt ? __int_as_float(0x7fc00000) : power_of_two(ek);
      a.cache.v_scale[scale_at] = power_of_two(ev);
    }
    if (mine) {
      uint8_t *k = k_codes + (held + group_of) * D, *v = v_codes + (held + group_of) * D;
      *reinterpret_cast<uint2*>(k + 8 * c) = codes8(k_lo, power_of_two(-ek));
      *reinterpret_cast<uint2*>(k + HALF + 8 * c) = codes8(k_hi, power_of_two(-ek));
      const uint2 a0 = codes8(v_lo, power_of_two(-ev)), a1 = codes8(v_hi, power_of_two(-ev));
      *reinterpret_cast<uint4*>(v + 16 * c) = make_uint4(a0.x, a0.y, a1.x, a1.y);
    }
  }
  store_queries(group_of);
  for (int from = group_of + AHEAD * TOKENS; from < n_units; from += AHEAD * TOKENS) {
    load_queries(from);
    store_queries(from);
  }
}

template <int D, typename T>
int launch(const AppendArgs& a, cudaStream_t stream) {
  launch_kernel(a.n_partials == 1 ? cache8_append_kernel<D, T, true> : cache8_append_kernel<D, T, false>, dim3(a.lists.n_writes, a.cache.kv_heads),
                TOKENS * (D / 16), 0, stream, a);
  return launch_status();
}

}  // namespace

// `qkv` (element type `in_dtype`): n_partials results partial_stride elements apart to be added in that order, each dense
// rows of (q_heads + 2 kv_heads) * head_dim.  The lists are those of llm_step_maps.  Rows of no request, and idle ones, are left as they
// were in q_out.  head_dim 64 or 128.
extern "C" int llm_cache8_append(const void* qkv, int in_dtype, int n_partials, long long partial_stride, void* q_out,
                                 const Cache8* cache, const StepLists* lists, const float* inv_freq, int q_heads, int write_cache,
                                 cudaStream_t stream) {
  if (lists->n_writes <= 0) return 0;
  const Cache8& c = *cache;
  if (c.kv_heads <= 0 || q_heads <= 0 || q_heads % c.kv_heads || c.kv_heads > 65535 || n_partials < 1 || c.page_tokens % SCALE_TOKENS ||
      c.page_tokens <= 0 || (c.head_dim != 64 && c.head_dim != 128))
    return ERR_BAD_SIZE;
  if (in_dtype != DT_F32 && in_dtype != DT_BF16) return ERR_BAD_DTYPE;
  const uintptr_t all = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(c.k) |
                        reinterpret_cast<uintptr_t>(c.v) | (uintptr_t)c.page_stride;
  if ((all & 15) || (n_partials > 1 && partial_stride % (in_dtype == DT_F32 ? 4 : 8))) return ERR_BAD_ALIGN;
  AppendArgs a{qkv, n_partials, partial_stride, reinterpret_cast<__nv_bfloat16*>(q_out), c, *lists, inv_freq, q_heads, write_cache};
  if (c.head_dim == 64) return in_dtype == DT_F32 ? launch<64, float>(a, stream) : launch<64, __nv_bfloat16>(a, stream);
  return in_dtype == DT_F32 ? launch<128, float>(a, stream) : launch<128, __nv_bfloat16>(a, stream);
}
