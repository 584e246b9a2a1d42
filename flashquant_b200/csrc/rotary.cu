// Rotary positions of the queries and keys of a step, and the same with the keys and values written to pages of
// 16-bit rows.  theta = position * frequency[j];  (a, b) -> scale (a cos - b sin, b cos + a sin), where the pair is
// (x_j, x_{j + R/2}) in the half layout and (x_2j, x_2j+1) in the interleaved one; values from R on are kept.
//
// Angles are taken in 64 bits: at position 10^6 an angle of 32 bits is off by 0.03.  In turns (position * frequency
// / 2 pi) the whole ones are dropped there, what is left goes through sincospif in 32 bits.
//
// Bound: HBM, every row is read and written once.  A CTA takes a few tokens: their angles go to shared memory
// once (the heads of a token share them), then every thread turns vectors of 16 bytes, all loads of a thread before
// its first store.
#include "fq_common.cuh"

namespace fq {

struct RotaryTensor {
  const void* src;
  void* dst;
  int64_t src_token, src_head, dst_token, dst_head;  // elements
  int heads;
};
struct RotaryArgs {
  RotaryTensor q, k, v;       // v: copied (append only)
  int64_t k_block, v_block;   // append: dst_token is the stride inside a block
  const void* positions;
  const void* slots;          // null: row i goes to row i
  const double* freq;
  int64_t tokens, num_slots;
  int head_dim, rotary_dim, block_size;
  int positions64, slots64;
  float scale, sign;
};

constexpr int kRotThreads = 256;

// (a cos - b sin, b cos + a sin), rounded the same way in every variant
__device__ __forceinline__ float2 turn(float a, float b, float2 cs) {
  return make_float2(__fmaf_rn(a, cs.x, -__fmul_rn(b, cs.y)), __fmaf_rn(b, cs.x, __fmul_rn(a, cs.y)));
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// N values to a vector; pairs of a work item: N in the half layout (two vectors), N / 2 or one in the other
template <typename T, int N, bool HALF>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs p, int per_cta) {
  extern __shared__ float2 angles[];  // [per_cta][rotary_dim / 2]
  __shared__ int64_t place[64];       // where a token's row goes; -1: nowhere
  const int tid = threadIdx.x;
  const int64_t token0 = int64_t(blockIdx.x) * per_cta;
  const int count = int(p.tokens - token0 < per_cta ? p.tokens - token0 : per_cta);
  const int half = p.rotary_dim / 2;

  auto position = [&](int64_t i) -> int64_t {
    return p.positions64 ? static_cast<const int64_t*>(p.positions)[i] : static_cast<const int32_t*>(p.positions)[i];
  };
  for (int i = tid; i < count * half; i += kRotThreads) {
    const int token = i / half, j = i - token * half;
    const double turns = double(position(token0 + token)) * (p.freq[j] * 0.15915494309189535);
    float s, c;
    sincospif(float(2.0 * (turns - rint(turns))), &s, &c);
    angles[i] = make_float2(c * p.scale, s * p.scale * p.sign);
  }
  for (int i = tid; i < count; i += kRotThreads) {
    int64_t to = token0 + i;
    if (p.positions && position(to) < 0) to = -1;  // (q and k of such a row are not touched)
    place[i] = to;
  }
  __syncthreads();

  const int pairs = HALF ? N : (N > 1 ? N / 2 : 1);
  const int turn_items = half / pairs;
  const int keep_items = (p.head_dim - p.rotary_dim) / N;
  const int items = turn_items + keep_items, all_items = p.head_dim / N;
  const int turned = (p.q.heads + p.k.heads) * items;
  const int total = turned + p.v.heads * all_items;
  for (int token = 0; token < count; ++token) {
    const int64_t from = token0 + token;
    int64_t slot = from;
    if (p.slots)
      slot = p.slots64 ? static_cast<const int64_t*>(p.slots)[from] : static_cast<const int32_t*>(p.slots)[from];
    const bool stored = !p.slots || (slot >= 0 && slot < p.num_slots);
    for (int i = tid; i < total; i += kRotThreads) {
      const bool is_v = i >= turned;
      const int per_head = is_v ? all_items : items;
      const int x = is_v ? i - turned : i;
      int head = x / per_head;
      const int item = x - head * per_head;
      const bool is_k = !is_v && head >= p.q.heads;
      if (is_k) head -= p.q.heads;
      const RotaryTensor& t = is_v ? p.v : (is_k ? p.k : p.q);
      if (!is_v && place[token] < 0) continue;
      if ((is_k || is_v) && !stored) continue;
      const T* src = static_cast<const T*>(t.src) + from * t.src_token + head * t.src_head;
      T* dst = static_cast<T*>(t.dst) + head * t.dst_head;
      if ((is_k || is_v) && p.slots)
        dst += slot / p.block_size * (is_v ? p.v_block : p.k_block) + slot % p.block_size * t.dst_token;
      else
        dst += from * t.dst_token;
      using V = Vec<T, N>;
      if (is_v || item >= turn_items) {
        const int at = is_v ? item * N : p.rotary_dim + (item - turn_items) * N;
        if (dst != src) *reinterpret_cast<V*>(dst + at) = *reinterpret_cast<const V*>(src + at);
        continue;
      }
      const float2* cs = angles + token * half + item * pairs;
      if constexpr (HALF) {
        V a = *reinterpret_cast<const V*>(src + item * N), b = *reinterpret_cast<const V*>(src + half + item * N);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float2 y = turn(to_f32(a.v[e]), to_f32(b.v[e]), cs[e]);
          a.v[e] = from_f32<T>(y.x);
          b.v[e] = from_f32<T>(y.y);
        }
        *reinterpret_cast<V*>(dst + item * N) = a;
        *reinterpret_cast<V*>(dst + half + item * N) = b;
      } else if constexpr (N > 1) {
        V a = *reinterpret_cast<const V*>(src + item * N);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 y = turn(to_f32(a.v[e]), to_f32(a.v[e + 1]), cs[e / 2]);
          a.v[e] = from_f32<T>(y.x);
          a.v[e + 1] = from_f32<T>(y.y);
        }
        *reinterpret_cast<V*>(dst + item * N) = a;
      } else {
        const float2 y = turn(to_f32(src[2 * item]), to_f32(src[2 * item + 1]), *cs);
        dst[2 * item] = from_f32<T>(y.x);
        dst[2 * item + 1] = from_f32<T>(y.y);
      }
    }
  }
}

static bool rows_aligned(const RotaryTensor& t, size_t size, bool src, bool dst) {
  return t.heads == 0 || ((!src || (aligned(t.src, 16) && (t.src_token | t.src_head) * int64_t(size) % 16 == 0)) &&
                          (!dst || (aligned(t.dst, 16) && (t.dst_token | t.dst_head) * int64_t(size) % 16 == 0)));
}

template <typename T>
static int launch_rotary(const RotaryArgs& p, bool half_layout, cudaStream_t stream) {
  constexpr int N = 16 / sizeof(T);
  const int per_cta = p.tokens <= 592 ? 1 : 4;
  const int64_t ctas = (p.tokens + per_cta - 1) / per_cta;
  FQ_REQUIRE(ctas <= 0x7fffffff, FQ_ERR_UNSUPPORTED, "rotary: too many tokens");
  const size_t smem = size_t(per_cta) * (p.rotary_dim / 2) * sizeof(float2);
  const bool wide = rows_aligned(p.q, sizeof(T), true, true) && rows_aligned(p.k, sizeof(T), true, true) &&
                    rows_aligned(p.v, sizeof(T), true, true) && (p.k_block | p.v_block) * int64_t(sizeof(T)) % 16 == 0 &&
                    p.head_dim % N == 0 && p.rotary_dim % (half_layout ? 2 * N : N) == 0;
  const dim3 grid = dim3(unsigned(ctas));
  if (wide && half_layout) rotary_kernel<T, N, true><<<grid, kRotThreads, smem, stream>>>(p, per_cta);
  else if (wide) rotary_kernel<T, N, false><<<grid, kRotThreads, smem, stream>>>(p, per_cta);
  else if (half_layout) rotary_kernel<T, 1, true><<<grid, kRotThreads, smem, stream>>>(p, per_cta);
  else rotary_kernel<T, 1, false><<<grid, kRotThreads, smem, stream>>>(p, per_cta);
  return check_launch("rotary");
}

static int rotary_common(const RotaryArgs& p, fq_dtype dtype, fq_rotary_layout layout, cudaStream_t stream) {
  const bool half = layout == FQ_ROTARY_HALF;
  switch (dtype) {
    case FQ_F32: return launch_rotary<float>(p, half, stream);
    case FQ_F16: return launch_rotary<__half>(p, half, stream);
    default: return launch_rotary<__nv_bfloat16>(p, half, stream);
  }
}

}  // namespace fq

using namespace fq;

static int rotary_check(fq_dtype dtype, int64_t tokens, int hq, int hkv, int head_dim, int rotary_dim,
                        fq_rotary_layout layout) {
  FQ_REQUIRE(tokens >= 0 && hq >= 0 && hkv >= 0 && rotary_dim >= 0, FQ_ERR_INVALID_ARGUMENT, "rotary: negative size");
  FQ_REQUIRE(dtype >= FQ_F32 && dtype <= FQ_BF16, FQ_ERR_INVALID_ARGUMENT, "rotary: unknown dtype");
  FQ_REQUIRE(layout == FQ_ROTARY_HALF || layout == FQ_ROTARY_INTERLEAVED, FQ_ERR_INVALID_ARGUMENT,
             "rotary: unknown layout");
  FQ_REQUIRE(head_dim > 0 && head_dim <= 1024 && rotary_dim <= head_dim && rotary_dim % 2 == 0, FQ_ERR_UNSUPPORTED,
             "rotary: the rotated part must be even and within a head of at most 1024 values (got %d of %d)", rotary_dim,
             head_dim);
  FQ_REQUIRE(hq <= 4096 && hkv <= 4096, FQ_ERR_UNSUPPORTED, "rotary: at most 4096 heads");
  return FQ_OK;
}

extern "C" int fq_rotary_embed(const void* q, const void* k, fq_dtype dtype, int64_t tokens, int num_q_heads,
                               int num_k_heads, int head_dim, int rotary_dim, const int64_t* strides,
                               const void* positions, int positions_are_int64, const double* frequencies,
                               fq_rotary_layout layout, float scale, int inverse, void* q_out, void* k_out,
                               fq_stream_t stream) {
  FQ_RANGE("fq_rotary_embed");
  if (const int rc = rotary_check(dtype, tokens, num_q_heads, num_k_heads, head_dim, rotary_dim, layout)) return rc;
  if (tokens == 0 || num_q_heads + num_k_heads == 0) return FQ_OK;
  FQ_REQUIRE(strides && positions && (rotary_dim == 0 || frequencies) && (num_q_heads == 0 || (q && q_out)) &&
                 (num_k_heads == 0 || (k && k_out)),
             FQ_ERR_INVALID_ARGUMENT, "rotary: null pointer");
  RotaryArgs p{};
  p.q = {q, q_out, strides[0], strides[1], strides[4], strides[5], num_q_heads};
  p.k = {k, k_out, strides[2], strides[3], strides[6], strides[7], num_k_heads};
  p.positions = positions;
  p.positions64 = positions_are_int64;
  p.freq = frequencies;
  p.tokens = tokens;
  p.head_dim = head_dim;
  p.rotary_dim = rotary_dim;
  p.scale = scale;
  p.sign = inverse ? -1.f : 1.f;
  return rotary_common(p, dtype, layout, stream);
}

extern "C" int fq_rotary_append_dense(const void* q, const void* key, const void* value, fq_dtype dtype, int64_t tokens,
                                      int num_q_heads, int num_kv_heads, int head_dim, int rotary_dim,
                                      const int64_t* strides, const void* positions, int positions_are_int64,
                                      const double* frequencies, fq_rotary_layout layout, float scale, void* q_out,
                                      void* key_cache, void* value_cache, int block_size, int64_t num_slots,
                                      const void* slot_mapping, int slots_are_int64, fq_stream_t stream) {
  FQ_RANGE("fq_rotary_append_dense");
  if (const int rc = rotary_check(dtype, tokens, num_q_heads, num_kv_heads, head_dim, rotary_dim, layout)) return rc;
  FQ_REQUIRE(dtype != FQ_F32, FQ_ERR_UNSUPPORTED, "dense append: pages are fp16 or bf16");
  FQ_REQUIRE(block_size > 0 && num_slots >= 0, FQ_ERR_INVALID_ARGUMENT, "dense append: bad cache size");
  if (tokens == 0 || num_q_heads + num_kv_heads == 0) return FQ_OK;
  FQ_REQUIRE(strides && (rotary_dim == 0 || (frequencies && positions)) && (num_q_heads == 0 || (q && q_out)) &&
                 (num_kv_heads == 0 || (key && value && key_cache && value_cache && slot_mapping)),
             FQ_ERR_INVALID_ARGUMENT, "dense append: null pointer");
  RotaryArgs p{};
  p.q = {q, q_out, strides[0], strides[1], strides[6], strides[7], num_q_heads};
  p.k = {key, key_cache, strides[2], strides[3], strides[9], strides[10], num_kv_heads};
  p.v = {value, value_cache, strides[4], strides[5], strides[12], strides[13], num_kv_heads};
  p.k_block = strides[8];
  p.v_block = strides[11];
  p.positions = positions;
  p.positions64 = positions_are_int64;
  p.slots = slot_mapping;
  p.slots64 = slots_are_int64;
  p.freq = frequencies;
  p.tokens = tokens;
  p.num_slots = num_slots;
  p.head_dim = head_dim;
  p.rotary_dim = rotary_dim;
  p.block_size = block_size;
  p.scale = scale;
  p.sign = 1.f;
  return rotary_common(p, dtype, layout, stream);
}
