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
// positions in registers (a thread eight entries of each of one token), so they are read once, and it alone
// settles the two scales: no atomics, no second pass.  The query heads that share the key/value head go through the same block:
// their angles are the ones the keys need, computed once into shared memory.
// Bound by memory for prompts (projections in, queries out), by its trips to memory for decoding steps.  One B200, a call after
// another from Python: 8 decoding requests (32 / 8 heads of 128) 13.2 us, 64 with three partial results (32 / 4 heads of 64) 13.6, a
// prompt's 2,048 tokens 23.6 (1.95 TB/s).

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

// Four neighbouring entries of the sum of the partial results.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, int n_partials, long long stride);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p, int n_partials, long long stride) {
  float4 v = *reinterpret_cast<const float4*>(p);
  for (int i = 1; i < n_partials; ++i) {
    const float4 w = *reinterpret_cast<const float4*>(p + i * stride);
    v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
  }
  return v;
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p, int n_partials, long long stride) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = 0; i < n_partials; ++i) {
    const uint2 raw = *reinterpret_cast<const uint2*>(p + i * stride);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
    v.x += a.x, v.y += a.y, v.z += b.x, v.w += b.y;
  }
  return v;
}

// (x, y) turned by the angles of `cs` = (cos, sin) pairs.
__device__ __forceinline__ void turn(float4& lo, float4& hi, const float2* cs) {
  const float4 a = lo, b = hi;
  lo = make_float4(a.x * cs[0].x - b.x * cs[0].y, a.y * cs[1].x - b.y * cs[1].y, a.z * cs[2].x - b.z * cs[2].y, a.w * cs[3].x - b.w * cs[3].y);
  hi = make_float4(b.x * cs[0].x + a.x * cs[0].y, b.y * cs[1].x + a.y * cs[1].y, b.z * cs[2].x + a.z * cs[2].y, b.w * cs[3].x + a.w * cs[3].y);
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The largest finite entry in size; `spoilt` if one is not finite, which then counts as zero.
__device__ __forceinline__ float largest_of(float4& x, bool& spoilt) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float& e = reinterpret_cast<float*>(&x)[i];
    if (!finite(e)) spoilt = true, e = 0.0f;
    m = fmaxf(m, fabsf(e));
  }
  return m;
}

// The smallest e with a <= 448 * 2^e = 1.75 * 2^(e + 8), within the bounds.
__device__ __forceinline__ int scale_exponent(float a) {
  const int bits = __float_as_int(a);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return min(max(e, SCALE_LEAST), SCALE_MOST);      // zero and numbers below the normal range: the least
}

__device__ __forceinline__ uint32_t codes4(float4 x, float factor) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x.x * factor, x.y * factor), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x.z * factor, x.w * factor), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float4 numbers4(uint32_t codes) {
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffff), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E4M3);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  return make_float4(x.x, x.y, y.x, y.y);
}

template <int D, typename T>
__global__ void __launch_bounds__(TOKENS * (D / 8)) cache8_append_kernel(const AppendArgs a) {
  constexpr int CHUNKS = D / 8, HALF = D / 2, THREADS = TOKENS * CHUNKS;
  pdl_launch_dependents();
  __shared__ float2 angles[TOKENS][HALF];
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
  const int page = page_of(a.cache, seq, first);
  const bool write = a.write_cache && page >= 0;
  const int in_page = first % a.cache.page_tokens;
  const long long at = (long long)page * a.cache.page_stride + ((long long)kvh * a.cache.page_tokens + in_page) * D;
  const long long scale_at = (long long)page * a.cache.scale_stride + (long long)kvh * (a.cache.page_tokens / TOKENS) + in_page / TOKENS;
  if (a.inv_freq) {
    // the angle's product in two parts, p f = hi + lo exactly, sin(hi + lo) = sin hi + lo cos hi: far positions keep their angle
    for (int i = tid; i < n_new * HALF; i += THREADS) {
      const float p = (float)(lo + i / HALF), f = a.inv_freq[i % HALF], hi = p * f, rest = fmaf(p, f, -hi);
      float s, co;
      sincosf(hi, &s, &co);
      angles[i / HALF][i % HALF] = make_float2(fmaf(-rest, s, co), fmaf(rest, co, s));
    }
  }
  __syncthreads();
  pdl_wait();

  const int group = a.q_heads / a.cache.kv_heads, n_heads = a.q_heads + 2 * a.cache.kv_heads;
  const T* qkv = reinterpret_cast<const T*>(a.qkv) + row0 * n_heads * D;
  // ---- keys and values: token `group_of` of the new ones; pairs 4 c .. 4 c + 3 of the key, entries 8 c .. 8 c + 7 of the value
  const bool mine = write && group_of < n_new;
  float4 k_lo, k_hi, v_lo, v_hi;
  k_lo = k_hi = v_lo = v_hi = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  bool spoilt = false;
  float k_most = 0.0f, v_most = 0.0f;
  if (mine) {
    const T* k = qkv + ((long long)group_of * n_heads + a.q_heads + kvh) * D;
    const T* v = k + (long long)a.cache.kv_heads * D;
    k_lo = load4<T>(k + 4 * c, a.n_partials, a.partial_stride);
    k_hi = load4<T>(k + HALF + 4 * c, a.n_partials, a.partial_stride);
    v_lo = load4<T>(v + 8 * c, a.n_partials, a.partial_stride);
    v_hi = load4<T>(v + 8 * c + 4, a.n_partials, a.partial_stride);
    if (a.inv_freq) turn(k_lo, k_hi, &angles[group_of][4 * c]);
    k_most = fmaxf(largest_of(k_lo, spoilt), largest_of(k_hi, spoilt));
    v_most = fmaxf(largest_of(v_lo, spoilt), largest_of(v_hi, spoilt));
  }
  if (write) {        // the same for every thread of the block
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
        if (ek > fk) {
          uint2* p = reinterpret_cast<uint2*>(k_codes + group_of * D + 8 * c);
          const uint2 old = *p;
          *p = make_uint2(codes4(numbers4(old.x), power_of_two(max(fk - ek, -126))), codes4(numbers4(old.y), power_of_two(max(fk - ek, -126))));
        }
        if (ev > fv) {
          uint2* p = reinterpret_cast<uint2*>(v_codes + group_of * D + 8 * c);
          const uint2 old = *p;
          *p = make_uint2(codes4(numbers4(old.x), power_of_two(max(fv - ev, -126))), codes4(numbers4(old.y), power_of_two(max(fv - ev, -126))));
        }
      }
    }
    if (tid == 0) {
      a.cache.k_scale[scale_at] = spoilt ? __int_as_float(0x7fc00000) : power_of_two(ek);
      a.cache.v_scale[scale_at] = power_of_two(ev);
    }
    if (mine) {
      uint8_t *k = k_codes + (held + group_of) * D, *v = v_codes + (held + group_of) * D;
      *reinterpret_cast<uint32_t*>(k + 4 * c) = codes4(k_lo, power_of_two(-ek));
      *reinterpret_cast<uint32_t*>(k + HALF + 4 * c) = codes4(k_hi, power_of_two(-ek));
      *reinterpret_cast<uint2*>(v + 8 * c) = make_uint2(codes4(v_lo, power_of_two(-ev)), codes4(v_hi, power_of_two(-ev)));
    }
  }
  // ---- the query heads of this key/value head: (head, token) pairs dealt to the groups of threads, tokens fastest, so that
  // a block with a single new token (a decoding request) turns up to 16 heads at once
  for (int u = group_of; u < n_new * group; u += TOKENS) {
    const int token = u % n_new, head = kvh * group + u / n_new;
    const T* q = qkv + ((long long)token * n_heads + head) * D;
    float4 lo4 = load4<T>(q + 4 * c, a.n_partials, a.partial_stride), hi4 = load4<T>(q + HALF + 4 * c, a.n_partials, a.partial_stride);
    if (a.inv_freq) turn(lo4, hi4, &angles[token][4 * c]);
    __nv_bfloat16* out = a.q_out + ((row0 + token) * a.q_heads + head) * D;
    const __nv_bfloat162 l0 = __floats2bfloat162_rn(lo4.x, lo4.y), l1 = __floats2bfloat162_rn(lo4.z, lo4.w);
    const __nv_bfloat162 h0 = __floats2bfloat162_rn(hi4.x, hi4.y), h1 = __floats2bfloat162_rn(hi4.z, hi4.w);
    *reinterpret_cast<uint2*>(out + 4 * c) = make_uint2(*reinterpret_cast<const uint32_t*>(&l0), *reinterpret_cast<const uint32_t*>(&l1));
    *reinterpret_cast<uint2*>(out + HALF + 4 * c) = make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
  }
}

template <int D, typename T>
int launch(const AppendArgs& a, cudaStream_t stream) {
  launch_kernel(cache8_append_kernel<D, T>, dim3(a.lists.n_writes, a.cache.kv_heads), TOKENS * (D / 8), 0, stream, a);
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
  if ((all & 15) || (n_partials > 1 && partial_stride % 4)) return ERR_BAD_ALIGN;
  AppendArgs a{qkv, n_partials, partial_stride, reinterpret_cast<__nv_bfloat16*>(q_out), c, *lists, inv_freq, q_heads, write_cache};
  if (c.head_dim == 64) return in_dtype == DT_F32 ? launch<64, float>(a, stream) : launch<64, __nv_bfloat16>(a, stream);
  return in_dtype == DT_F32 ? launch<128, float>(a, stream) : launch<128, __nv_bfloat16>(a, stream);
}
