// Rotary positions of the queries and keys of a step, and the same with the keys and values written to pages of
// 16-bit rows.  theta = position * frequency[j];  (a, b) -> scale (a cos - b sin, b cos + a sin), where the pair is
// (x_j, x_{j + R/2}) in the half layout and (x_2j, x_2j+1) in the interleaved one; values from R on are kept.
//
// Angles are taken in 64 bits: at position 10^6 an angle of 32 bits is off by 0.03.  In turns (position * frequency
// / 2 pi) the whole ones are dropped there, what is left goes through sincospif in 32 bits.
//
// Bound: HBM, every row is read and written once.  As many CTAs as there is room for go through the tokens, a few at a
// time.  Each time they find what the heads of those tokens share, the angles and where their rows in the pages are,
// in shared memory.  Every warp has a job, some heads of q, k or v: which tensor it works on is the same for all its
// lanes, a lane keeps its place (16 bytes, or two times 16 that make pairs) in the same rows of each token, goes on by a
// stride, and has the next token's on the way before it stores this one's, the next angles being found meanwhile.
// (With rows of all three tensors dealt to the threads of a CTA the same work took 240 instructions to a place and
// three times as long.)
//
// Measured, 32 / 8 heads of 128, bf16: 32 tokens 3.1 us, with the append 3.4; 8192 tokens 31.2 us, 37.5 with it: 5.4 TB/s
// read and written, 82 % of a copy (16384 tokens: 89 %); the loads that 30 warps of an SM have under way bound it.  Rows that
// are not whole vectors of 16 bytes go value by value: 8192 tokens of 96 values, 48 of them rotated 28.1 us, 24 of them 67.6.
#include <algorithm>

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

constexpr int kRotWarps = 8;   // of a CTA at most
constexpr int kRotTokens = 4;  // at a time, at most

// (a cos - b sin, b cos + a sin), rounded the same way in every variant
__device__ __forceinline__ float2 turn(float a, float b, float2 cs) {
  return make_float2(__fmaf_rn(a, cs.x, -__fmul_rn(b, cs.y)), __fmaf_rn(b, cs.x, __fmul_rn(a, cs.y)));
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

struct RotaryPlace {
  int64_t k, v;         // append: offsets of the token's rows
  bool placed, stored;  // its position is not negative; it has a slot
};

// The jobs of a tensor: `rows` rows to a lane, 32 / places side by side, further jobs for places beyond 32.
struct RotaryJobs {
  int places, side, parts, count;
  __host__ __device__ RotaryJobs(int all, int heads, int rows)
      : places(all < 32 ? all : 32), side(32 / places), parts((all + 31) / 32),
        count((heads + rows * side - 1) / (rows * side) * parts) {}
};
// The values of a place stand in one vector or in two: of a part that is turned the two of its pairs, of one that is kept
// two that are half of it apart.  Places of a part of `values`:
__host__ __device__ inline bool rotary_two(int n, bool half_layout) { return half_layout || n == 1; }
__host__ __device__ inline int rotary_kept(int n, bool half_layout, int values) {
  return values / (rotary_two(n, half_layout) && values % (2 * n) == 0 ? 2 * n : n);
}
__host__ __device__ inline int rotary_places(int n, bool half_layout, int head_dim, int rotary_dim) {
  return rotary_dim / (rotary_two(n, half_layout) ? 2 * n : n) + rotary_kept(n, half_layout, head_dim - rotary_dim);
}
__host__ __device__ inline int rotary_rows(int n, bool half_layout) { return rotary_two(n, half_layout) ? 2 : 4; }

// values 2 k and 2 k + 1 of a vector
template <typename T, int N>
__device__ __forceinline__ float2 get2(const Vec<T, N>& x, int k) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(x.v[2 * k], x.v[2 * k + 1]);
  } else {
    float y[2];
    load2(x.v + 2 * k, y);
    return make_float2(y[0], y[1]);
  }
}
__device__ __forceinline__ void put2(float* at, float x, float y) { at[0] = x; at[1] = y; }
__device__ __forceinline__ void put2(__half* at, float x, float y) {
  *reinterpret_cast<__half2*>(at) = __floats2half2_rn(x, y);
}
__device__ __forceinline__ void put2(__nv_bfloat16* at, float x, float y) {
  *reinterpret_cast<__nv_bfloat162*>(at) = __floats2bfloat162_rn(x, y);
}

// N values to a vector.  HALF: pairs half a rotated part apart, else adjacent.
template <typename T, int N, bool HALF>
__global__ void __launch_bounds__(kRotWarps * 32, 4) rotary_kernel(const RotaryArgs p, int batch) {
  using V = Vec<T, N>;
  constexpr int kPairs = HALF ? N : (N > 1 ? N / 2 : 1), kRows = HALF || N == 1 ? 2 : 4;
  constexpr bool kTwo = HALF || N == 1;  // the values of a place stand in two vectors
  // [2][batch][chunk][place][2]: the cosines and sines of a place are read two at a time, adjacent places together
  extern __shared__ __align__(16) float2 angles[];
  constexpr int kChunk = kPairs > 1 ? 2 : 1;
  __shared__ RotaryPlace where[2][kRotTokens];
  const int half = p.rotary_dim / 2, turns_of = half / kPairs;
  const int tid = threadIdx.x, lane = tid & 31;
  auto integer = [](const void* x, int wide, int64_t i) -> int64_t {
    return wide ? static_cast<const int64_t*>(x)[i] : static_cast<const int32_t*>(x)[i];
  };
  auto prepare = [&](int64_t token0, int count, int buffer) {
    for (int i = tid; i < half * count; i += blockDim.x) {
      const int of = i / half, j = i - of * half;
      const double turns = double(integer(p.positions, p.positions64, token0 + of)) * (p.freq[j] * 0.15915494309189535);
      float s, c;
      sincospif(float(2.0 * (turns - rint(turns))), &s, &c);
      const int place = j / kPairs, e = j % kPairs;
      angles[(buffer * batch + of) * half + (e / kChunk * turns_of + place) * kChunk + e % kChunk] =
          make_float2(c * p.scale, s * p.scale * p.sign);
    }
    if (tid < count) {
      RotaryPlace w{0, 0, true, true};
      if (p.positions) w.placed = integer(p.positions, p.positions64, token0 + tid) >= 0;
      if (p.slots) {
        const int64_t slot = integer(p.slots, p.slots64, token0 + tid);
        w.stored = slot >= 0 && slot < p.num_slots;
        const int64_t block = w.stored ? slot / p.block_size : 0, row = w.stored ? slot - block * p.block_size : 0;
        w.k = block * p.k_block + row * p.k.dst_token;
        w.v = block * p.v_block + row * p.v.dst_token;
      }
      where[buffer][tid] = w;
    }
  };

  // ---- this warp's job ---------------------------------------------------------------------------------
  const int all = rotary_places(N, HALF, p.head_dim, p.rotary_dim);
  const int all_v = rotary_kept(N, HALF, p.head_dim);
  const RotaryJobs jq(all, p.q.heads, kRows), jk(all, p.k.heads, kRows), jv(all_v, p.v.heads, kRows);
  int job = blockIdx.y * (blockDim.x / 32) + __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int kind = job < jq.count ? 0 : (job < jq.count + jk.count ? 1 : 2);
  if (kind > 0) job -= jq.count;
  if (kind > 1) job -= jk.count;
  const RotaryTensor& t = kind == 2 ? p.v : (kind == 1 ? p.k : p.q);
  const RotaryJobs& j = kind == 2 ? jv : (kind == 1 ? jk : jq);
  const bool working = job < j.count;
  const int row = lane / j.places, place = job % j.parts * 32 + lane - row * j.places;
  const int head = job / j.parts * kRows * j.side + row;
  const bool turned = kind < 2 && place < turns_of;
  const int kept = kind == 2 ? p.head_dim : p.head_dim - p.rotary_dim;
  const bool two = kTwo && (turned || kept % (2 * N) == 0);
  const int rows = !working || row >= j.side || place >= (kind == 2 ? all_v : all) || head >= t.heads
                       ? 0
                       : min(kRows, (t.heads - head + j.side - 1) / j.side);
  int at = place * N, too = 0;  // the values of a place; how far its second vector is behind the first
  if (!turned) {
    if (kind < 2) at += p.rotary_dim - turns_of * N;
    too = kept / 2;
  } else if (kTwo) {
    if (!HALF) at = 2 * place;
    too = HALF ? half : 1;
  }
  const bool paged = p.slots && kind > 0;
  const T* const src = static_cast<const T*>(t.src) + head * t.src_head + at;
  T* const dst = static_cast<T*>(t.dst) + head * t.dst_head + at;
  const int64_t src_row = j.side * t.src_head, dst_row = j.side * t.dst_head;

  V a[kRows], b[kTwo ? kRows : 1];
  auto load = [&](int64_t token, V (&u)[kRows], V (&w)[kTwo ? kRows : 1]) {
    const T* x = src + token * t.src_token;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r >= rows) break;
      u[r] = *reinterpret_cast<const V*>(x + r * src_row);
      if (kTwo && two) w[r] = *reinterpret_cast<const V*>(x + r * src_row + too);
    }
  };
  const int64_t step = int64_t(gridDim.x) * batch;
  int64_t token0 = int64_t(blockIdx.x) * batch;
  if (token0 < p.tokens) load(token0, a, b);
  for (int buffer = 0; token0 < p.tokens; token0 += step, buffer ^= 1) {
    const int count = int(p.tokens - token0 < batch ? p.tokens - token0 : batch);
    prepare(token0, count, buffer);
    __syncthreads();
    for (int i = 0; i < count; ++i) {
      V next_a[kRows], next_b[kTwo ? kRows : 1];
      const int64_t next = i + 1 < count ? token0 + i + 1 : token0 + step;
      if (next < p.tokens) load(next, next_a, next_b);
      const RotaryPlace& w = where[buffer][i];
      if ((kind == 2 || w.placed) && (kind == 0 || w.stored)) {
        if (turned) {
          float2 cs[kPairs];
          const float2* c = angles + (buffer * batch + i) * half + place * kChunk;
#pragma unroll
          for (int e = 0; e < kPairs; e += kChunk) {
            if constexpr (kChunk == 2) {
              const float4 x = *reinterpret_cast<const float4*>(c + e * turns_of);
              cs[e] = make_float2(x.x, x.y);
              cs[e + 1] = make_float2(x.z, x.w);
            } else {
              cs[e] = c[e * turns_of];
            }
          }
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            if constexpr (N == 1) {
              const float2 y = turn(to_f32(a[r].v[0]), to_f32(b[r].v[0]), cs[0]);
              a[r].v[0] = from_f32<T>(y.x);
              b[r].v[0] = from_f32<T>(y.y);
            } else if constexpr (HALF) {
#pragma unroll
              for (int k = 0; k < N / 2; ++k) {
                const float2 u = get2(a[r], k), v = get2(b[r], k);
                const float2 y = turn(u.x, v.x, cs[2 * k]), z = turn(u.y, v.y, cs[2 * k + 1]);
                put2(a[r].v + 2 * k, y.x, z.x);
                put2(b[r].v + 2 * k, y.y, z.y);
              }
            } else {
#pragma unroll
              for (int k = 0; k < N / 2; ++k) {
                const float2 u = get2(a[r], k), y = turn(u.x, u.y, cs[k]);
                put2(a[r].v + 2 * k, y.x, y.y);
              }
            }
          }
        }
        T* y = dst + (paged ? (kind == 2 ? w.v : w.k) : (token0 + i) * t.dst_token);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          if (r >= rows) break;
          *reinterpret_cast<V*>(y + r * dst_row) = a[r];
          if (kTwo && two) *reinterpret_cast<V*>(y + r * dst_row + too) = b[r];
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        a[r] = next_a[r];
        if (kTwo) b[r] = next_b[r];
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
  const bool wide = rows_aligned(p.q, sizeof(T), true, true) && rows_aligned(p.k, sizeof(T), true, true) &&
                    rows_aligned(p.v, sizeof(T), true, true) && (p.k_block | p.v_block) * int64_t(sizeof(T)) % 16 == 0 &&
                    p.head_dim % N == 0 && p.rotary_dim % (half_layout ? 2 * N : N) == 0;
  const int n = wide ? N : 1, rows = rotary_rows(n, half_layout);
  const int all = rotary_places(n, half_layout, p.head_dim, p.rotary_dim);
  const int all_v = rotary_kept(n, half_layout, p.head_dim);
  const int jobs = RotaryJobs(all, p.q.heads, rows).count + RotaryJobs(all, p.k.heads, rows).count +
                   RotaryJobs(all_v, p.v.heads, rows).count;
  const int groups = (jobs + kRotWarps - 1) / kRotWarps, warps = (jobs + groups - 1) / groups;
  const auto kernel = wide ? (half_layout ? rotary_kernel<T, N, true> : rotary_kernel<T, N, false>)
                           : (half_layout ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>);
  const auto smem = [&](int batch) { return 2 * size_t(batch) * (p.rotary_dim / 2) * sizeof(float2); };
  // One token at a time as long as each has CTAs of its own that are all resident (bf16, 1 and 2 at a time: 40 heads of 128, 888
  // resident, 700 tokens 5.7, 6.3 us, 800: 6.2, 6.5, 1000: 7.3, 7.2; 72 heads, 444: 420 tokens 6.1, 6.3, 450: 6.9, 6.6, 592: 8.0,
  // 7.3; 40 heads with the append, 740: 740 tokens 6.6, 6.7, 800: 7.5, 6.9; 32 of 64, 2368: 1184 tokens 5.1, 5.6, 2300: 7.2, 6.9).
  int batch = 1;
  int64_t ctas = p.tokens;
  if (ctas > 64) {  // no more CTAs than are resident together
    int device = 0, sms = 0, fit = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, warps * 32, smem(kRotTokens));
    if (e != cudaSuccess) return fail(FQ_ERR_CUDA, "rotary: %s", cudaGetErrorString(e));
    const int64_t most = std::max(1, sms * fit / groups);
    if (p.tokens > most) batch = 2;
    if (batch == 2 && p.tokens > 1184) {
      // what leaves the last round of the CTAs fullest, a token less at a time counted as 2 % more work (8192 tokens:
      // 31.7 us with 4, 30.6 with 3; of heads of 64 19.6 and 18.4)
      int64_t least = INT64_MAX;
      for (int n = kRotTokens; n > 1; --n) {
        const int64_t rounds = ((p.tokens + n - 1) / n + most - 1) / most, cost = rounds * n * (50 + kRotTokens - n);
        if (cost < least) {
          least = cost;
          batch = n;
        }
      }
    }
    ctas = std::min((p.tokens + batch - 1) / batch, most);
  }
  kernel<<<dim3(unsigned(ctas), groups), warps * 32, smem(batch), stream>>>(p, batch);
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
