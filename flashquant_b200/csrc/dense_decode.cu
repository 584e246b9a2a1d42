// Attention of one new token per sequence over pages of 16-bit keys and values, split over the length of
// the cache and joined.  o_h = sum_t softmax_t(scale q_h k_t) v_t over the last `window` of the sequence's tokens.
//
// Bound: HBM.  4 D bytes per (token, KV head) against 4 D (query heads per KV head) operations: at most 16
// operations a byte here, a thirtieth of what the tensor pipe would need to be the limit.  So the products run
// on mma.sync (16 x 8 x 16, an 8- or 16-row query block as the A operand), whose operands come straight from the
// rows that cp.async has laid down; tcgen05 with its 128 rows would be idle in nine tenths of them.
//
// Every warp streams on its own: a ring of tiles of 16 tokens in shared memory, filled by cp.async (16 bytes a
// lane, rows outside the sequence filled with zeros), no barrier of the CTA in the loop.  How the tiles are dealt
// out: dense_split.h.  Sums, maxima and weights are fp32; a weight enters the value product as two 16-bit terms
// (hi + lo, 2^-17 of it or better), so that the output is rounded once, at the end.  With up to eight query heads
// per unit the lo terms are the rows 8..15 of the A operand and cost nothing.
#include <algorithm>
#include <type_traits>

#include "dense_split.h"
#include "fq_common.cuh"

namespace fq {

constexpr int kDenseMaxCtas = 148;
constexpr int kDenseMaxSeqs = 2048;
constexpr size_t kDenseHead = 32768;     // status word, counters (zero between calls); then the pieces
constexpr size_t kDenseCounters = 256;   // [CTA][warp]
constexpr int kDenseShortest = 4;        // tiles to a run at least

struct DenseArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int32_t *table, *lens;
  int64_t q_seq, q_head;                 // strides, in elements
  int64_t k_block, k_token, k_head, v_block, v_token, v_head;
  int64_t table_stride, num_blocks;
  int seqs, hq, hkv, table_width, block_size, window;
  int chunks, rows;                      // units of a KV head, query heads of a unit
  int side, piece_floats;                // units side by side; stride of the pieces
  float scale_log2;
  uint32_t* status;
  uint32_t* counters;
  float* pieces;
};

template <int D>
struct DenseShape {
  static constexpr int kWarps = D > 128 ? 4 : 8;
  static constexpr int kPitch = 2 * D + 16;  // bytes of a row: 16 beyond it, so that 8 rows fall into all banks
  static constexpr int kTensor = kDenseTile * kPitch;
  static constexpr int kStage = 2 * kTensor;
  static constexpr int kStages = D == 64 ? 5 : (D == 96 ? 4 : 3);
  static constexpr int kRing = kStages * kStage;
  static constexpr int kSmem = kWarps * kRing;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}

template <typename T>
struct Dense16;
template <>
struct Dense16<__half> {
  // fp16 weights: 2^14 times the weight, so that the small ones keep their digits
  static constexpr float kLift = 14.f;
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_f16(c, a[0], a[1], a[2], a[3], b0, b1);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) { return pack_half2(x, y); }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  }
};
template <>
struct Dense16<__nv_bfloat16> {
  static constexpr float kLift = 0.f;
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16(c, a[0], a[1], a[2], a[3], b0, b1);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};

// Where a warp stands in the list of tiles.
struct DenseCursor {
  int at, end;        // entries of its run
  int a, b;           // entries of the unit group
  int seq, group;     // the sequence, its unit group
  int begin, len;     // tokens seen: [begin, len)
  int tile;           // of the sequence
};

template <typename T, int D, bool R16>
__global__ void __launch_bounds__(DenseShape<D>::kWarps * 32, 1) dense_decode_kernel(const DenseArgs p) {
  using S = DenseShape<D>;
  using X = Dense16<T>;
  constexpr int kRows = R16 ? 16 : 8;
  constexpr int kSteps = D / 16, kBlocks = D / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int warp_total[S::kWarps];
  int* const prefix = reinterpret_cast<int*>(smem + S::kSmem);  // [seqs + 1]
  int* const lengths = prefix + p.seqs + 1;                     // [seqs]
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int g = lane >> 2, t = lane & 3;
  const int64_t room = int64_t(p.table_width) * p.block_size;
  const int unit_groups = p.hkv * p.chunks / p.side;

  // ---- the list: prefix sums of the sequences' tiles -------------------------------------------------
  {
    const int each = (p.seqs + S::kWarps * 32 - 1) / (S::kWarps * 32);
    const int s0 = min(tid * each, p.seqs), s1 = min(s0 + each, p.seqs);
    int sum = 0;
    for (int s = s0; s < s1; ++s) {
      const int given = p.lens[s];
      const DenseSpan span = dense_span(given, room, p.window);
      if (given > span.len && blockIdx.x == 0) atomicOr(p.status, FQ_DEV_BAD_BLOCK_INDEX);
      lengths[s] = span.len;
      sum += span.tiles * unit_groups;
      prefix[s + 1] = sum;
    }
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    if (lane == 31) warp_total[warp] = before;
    before -= sum;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before += warp_total[w];
    if (tid == 0) prefix[0] = 0;
    for (int s = s0; s < s1; ++s) prefix[s + 1] += before;
    __syncthreads();
  }
  const int teams = S::kWarps / p.side;
  const int team = warp / p.side, member = warp - team * p.side;
  const DenseCut cut = dense_cut(prefix[p.seqs], gridDim.x, teams, kDenseShortest);

  // rows of sequences without a token
  for (int s = blockIdx.x; s < p.seqs; s += gridDim.x) {
    if (prefix[s + 1] != prefix[s]) continue;
    uint32_t* o = static_cast<uint32_t*>(p.out) + int64_t(s) * p.hq * (D / 2);
    for (int i = tid; i < p.hq * (D / 2); i += S::kWarps * 32) o[i] = 0u;
    if (p.lse)
      for (int i = tid; i < p.hq; i += S::kWarps * 32) p.lse[int64_t(s) * p.hq + i] = -INFINITY;
  }

  // ---- cursors ----------------------------------------------------------------------------------------
  auto enter = [&](DenseCursor& c) {  // c.seq, c.group -> the other fields, at the unit group's first entry
    c.len = lengths[c.seq];
    const DenseSpan span = dense_span(c.len, room, p.window);
    c.begin = span.begin;
    c.a = prefix[c.seq] + c.group * span.tiles;
    c.b = c.a + span.tiles;
    c.tile = span.first_tile;
  };
  auto start = [&](DenseCursor& c, int run) {
    c.at = cut.begin(run);
    c.end = cut.end(run);
    if (c.at >= c.end) return;
    int lo = 0, hi = p.seqs - 1;  // the sequence whose entries hold c.at
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid + 1] > c.at) hi = mid; else lo = mid + 1;
    }
    c.seq = lo;
    const int tiles = (prefix[lo + 1] - prefix[lo]) / unit_groups;
    c.group = (c.at - prefix[lo]) / tiles;
    enter(c);
    c.tile += c.at - c.a;
  };
  auto advance = [&](DenseCursor& c) {
    ++c.at;
    ++c.tile;
    if (c.at < c.b || c.at >= c.end) return;
    if (++c.group == unit_groups) {
      c.group = 0;
      do ++c.seq; while (prefix[c.seq + 1] == prefix[c.seq]);
    }
    enter(c);
  };

  const int run = blockIdx.x * teams + team;
  const uint32_t ring = smem_u32(smem) + warp * S::kRing;
  const int tiles_per_block = p.block_size / kDenseTile;

  DenseCursor ld;
  start(ld, run);
  DenseCursor cu = ld;
  int block = 0;  // the page of ld's tile (loaded a tile ahead of its use)
  auto look_up = [&] {
    if (ld.at < ld.end) block = p.table[ld.seq * p.table_stride + ld.tile / tiles_per_block];
  };
  look_up();
  uint32_t bad = 0;  // bit i: stage i holds a tile whose page does not exist
  auto issue = [&](int stage) {
    if (ld.at < ld.end) {
      const bool ok = unsigned(block) < uint64_t(p.num_blocks);
      bad = ok ? bad & ~(1u << stage) : bad | (1u << stage);
      const int first = ld.tile * kDenseTile;
      const int head = (ld.group * p.side + member) / p.chunks;
      const int64_t id = ok ? block : 0;
      const int row = (ld.tile % tiles_per_block) * kDenseTile;
      const T* k = static_cast<const T*>(p.k) + id * p.k_block + row * p.k_token + head * p.k_head;
      const T* v = static_cast<const T*>(p.v) + id * p.v_block + row * p.v_token + head * p.v_head;
      const int lo = ld.begin - first, hi = ok ? ld.len - first : 0;
      const uint32_t dst = ring + stage * S::kStage;
      constexpr int kPerRow = D / 8;
#pragma unroll
      for (int c = 0; c < kDenseTile * kPerRow / 32; ++c) {
        const int i = lane + 32 * c, r = i / kPerRow, col = i % kPerRow;
        const bool valid = r >= lo && r < hi;
        const int64_t rr = valid ? r : 0;
        cp_async16(dst + r * S::kPitch + col * 16, k + (valid ? rr * p.k_token + col * 8 : 0), valid);
        cp_async16(dst + S::kTensor + r * S::kPitch + col * 16, v + (valid ? rr * p.v_token + col * 8 : 0),
                   valid);
      }
      advance(ld);
      look_up();
    }
    cp_async_commit();
  };

  // ---- state of the unit in work ----------------------------------------------------------------------
  uint32_t qf[kSteps][R16 ? 4 : 2];
  float acc[kBlocks][4];
  float top[R16 ? 2 : 1], sum[R16 ? 2 : 1];

  auto unit_heads = [&](const DenseCursor& c, int& head0, int& count) {
    const int unit = c.group * p.side + member, group = p.hq / p.hkv;
    const int kv = unit / p.chunks, chunk = unit - kv * p.chunks;
    head0 = kv * group + chunk * p.rows;
    count = min(p.rows, group - chunk * p.rows);
  };
  auto begin_unit = [&] {
    int head0, count;
    unit_heads(cu, head0, count);
    const T* q = static_cast<const T*>(p.q) + cu.seq * p.q_seq + head0 * p.q_head;
#pragma unroll
    for (int r = 0; r < (R16 ? 2 : 1); ++r) {
      const bool real = g + 8 * r < count;
      const T* row = q + (real ? (g + 8 * r) * p.q_head : 0) + 2 * t;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(row + 16 * s);
        const uint32_t y = *reinterpret_cast<const uint32_t*>(row + 16 * s + 8);
        qf[s][r] = real ? x : 0u;
        qf[s][(R16 ? 2 : 1) + r] = real ? y : 0u;
      }
      top[r] = -INFINITY;
      sum[r] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  };

  auto tile_step = [&](int stage) {
    const uint32_t kt = ring + stage * S::kStage, vt = kt + S::kTensor;
    const int mid = lane >> 3;
    // scores: rows = heads, columns = tokens (two blocks of eight)
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    const uint32_t ka = kt + ((mid >> 1) * 8 + (lane & 7)) * S::kPitch + (mid & 1) * 16;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      uint32_t b[4];
      ldmatrix4(b, ka + i * 32);
      uint32_t a[4];
      if constexpr (R16) {
        a[0] = qf[i][0]; a[1] = qf[i][1]; a[2] = qf[i][2]; a[3] = qf[i][3];
      } else {
        a[0] = qf[i][0]; a[1] = 0u; a[2] = qf[i][1]; a[3] = 0u;
      }
      X::mma(s[0], a, b[0], b[1]);
      X::mma(s[1], a, b[2], b[3]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] *= p.scale_log2;
    const int first = cu.tile * kDenseTile;
    const int lo = cu.begin - first, hi = (bad >> stage) & 1 ? 0 : cu.len - first;
    if (lo > 0 || hi < kDenseTile) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = n * 8 + 2 * t + (e & 1);
          if (at < lo || at >= hi) s[n][e] = -INFINITY;
        }
    }
    uint32_t hi_a[4], lo_a[4];
#pragma unroll
    for (int r = 0; r < (R16 ? 2 : 1); ++r) {
      float m = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const float now = fmaxf(top[r], m);
      const float ref = now == -INFINITY ? 0.f : now;
      if (__any_sync(0xffffffffu, now != top[r])) {
        const float f = fast_exp2(top[r] - ref);
        sum[r] *= f;
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
          acc[j][2 * r] *= f;
          acc[j][2 * r + 1] *= f;
          if constexpr (!R16) {
            acc[j][2] *= f;
            acc[j][3] *= f;
          }
        }
        top[r] = now;
      }
      const float shift = X::kLift - ref;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float x = fast_exp2(s[n][2 * r] + shift);
        const float y = fast_exp2(s[n][2 * r + 1] + shift);
        sum[r] += x + y;
        const uint32_t h = X::pack(x, y);
        const float2 back = X::unpack(h);
        const uint32_t l = X::pack(x - back.x, y - back.y);
        if constexpr (R16) {
          hi_a[2 * n + r] = h;
          lo_a[2 * n + r] = l;
        } else {
          hi_a[2 * n] = h;
          hi_a[2 * n + 1] = l;
        }
      }
    }
    const uint32_t va = vt + ((mid & 1) * 8 + (lane & 7)) * S::kPitch + (mid >> 1) * 16;
#pragma unroll
    for (int j = 0; j < kBlocks; j += 2) {
      uint32_t b[4];
      ldmatrix4_trans(b, va + j * 16);
      X::mma(acc[j], hi_a, b[0], b[1]);
      X::mma(acc[j + 1], hi_a, b[2], b[3]);
      if constexpr (R16) {
        X::mma(acc[j], lo_a, b[0], b[1]);
        X::mma(acc[j + 1], lo_a, b[2], b[3]);
      }
    }
  };

  // ---- results ----------------------------------------------------------------------------------------
  auto piece_of = [&](int run_, int slot) {
    return p.pieces + ((int64_t(run_) * p.side + member) * 2 + slot) * p.piece_floats;
  };
  auto write_pair = [&](int seq, int head, int dim, float x, float y) {
    *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (int64_t(seq) * p.hq + head) * D + dim) = X::pack(x, y);
  };
  auto write_lse = [&](int seq, int head, float m, float l) {
    if (p.lse)
      p.lse[int64_t(seq) * p.hq + head] = l == 0.f ? -INFINITY : (m + log2f(l) - X::kLift) * 0.69314718f;
  };
  // the warp's unit: to `out` (dst null), or as a piece [rows][D], [rows][2] (maximum, sum)
  auto flush = [&](float* dst) {
    int head0, count;
    unit_heads(cu, head0, count);
#pragma unroll
    for (int r = 0; r < (R16 ? 2 : 1); ++r) {
      float l = sum[r];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const int row = g + 8 * r;
      if (row >= count) continue;
      const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        float x = acc[j][2 * r], y = acc[j][2 * r + 1];
        if constexpr (!R16) {  // the lo terms
          x += acc[j][2];
          y += acc[j][3];
        }
        if (dst)
          *reinterpret_cast<float2*>(dst + row * D + 8 * j + 2 * t) = make_float2(x, y);
        else
          write_pair(cu.seq, head0 + row, 8 * j + 2 * t, x * f, y * f);
      }
      if (t == 0) {
        if (dst)
          *reinterpret_cast<float2*>(dst + p.rows * D + 2 * row) = make_float2(top[r], l);
        else
          write_lse(cu.seq, head0 + row, top[r], l);
      }
    }
  };

  // Joins n pieces (piece(i): the i-th; SHARED: in shared memory, else in the workspace) into `out` or one
  // piece.  32 at a time: lane r finds the weights of row r and leaves them in the warp's part of shared memory,
  // then every lane sums its columns of four dimensions.
  float* const weights = reinterpret_cast<float*>(smem + warp * S::kRing);  // [33][kRows]
  float* const meet = weights + 33 * kRows;                                 // a piece, of a merging CTA
  auto join = [&](auto shared, const DenseCursor& c, int n, auto piece, float* dst) {
    constexpr bool kShared = decltype(shared)::value;
    auto load2 = [](const float* x) {
      const float2* y = reinterpret_cast<const float2*>(x);
      if constexpr (kShared) return *y; else return __ldcg(y);
    };
    auto load4 = [](const float* x) {
      const float4* y = reinterpret_cast<const float4*>(x);
      if constexpr (kShared) return *y; else return __ldcg(y);
    };
    int head0, count;
    unit_heads(c, head0, count);
    constexpr int kVecs = kRows * D / 4 / 32;  // columns of a lane
    float4 o[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;  // of row `lane`
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int some = min(32, n - i0);
      __syncwarp();
      if (lane < count) {
        float now = m;
        for (int i = 0; i < some; ++i) now = fmaxf(now, load2(piece(i0 + i) + p.rows * D + 2 * lane).x);
        const float ref = now == -INFINITY ? 0.f : now;
        const float f = fast_exp2(m - ref);
        l *= f;
        for (int i = 0; i < some; ++i) {
          const float2 x = load2(piece(i0 + i) + p.rows * D + 2 * lane);
          const float w = fast_exp2(x.x - ref);
          l = fmaf(w, x.y, l);
          weights[i * kRows + lane] = w;
        }
        m = now;
        weights[32 * kRows + lane] = f;
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int row = (lane + 32 * i) * 4 / D;
        const float f = row < count ? weights[32 * kRows + row] : 0.f;
        o[i].x *= f; o[i].y *= f; o[i].z *= f; o[i].w *= f;
      }
#pragma unroll 4
      for (int k = 0; k < some; ++k) {
        const float* src = piece(i0 + k);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const int row = (lane + 32 * i) * 4 / D;
          if (row < count) {
            const float w = weights[k * kRows + row];
            const float4 x = load4(src + 4 * (lane + 32 * i));
            o[i].x = fmaf(w, x.x, o[i].x);
            o[i].y = fmaf(w, x.y, o[i].y);
            o[i].z = fmaf(w, x.z, o[i].z);
            o[i].w = fmaf(w, x.w, o[i].w);
          }
        }
      }
    }
    __syncwarp();
    if (lane < count) {
      if (dst)
        *reinterpret_cast<float2*>(dst + p.rows * D + 2 * lane) = make_float2(m, l);
      else
        write_lse(c.seq, head0 + lane, m, l);
      weights[lane] = l == 0.f ? 0.f : 1.f / l;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int row = (lane + 32 * i) * 4 / D, dim = (lane + 32 * i) * 4 % D;
      if (row >= count) continue;
      if (dst) {
        reinterpret_cast<float4*>(dst)[lane + 32 * i] = o[i];
      } else {
        const float f = weights[row];
        write_pair(c.seq, head0 + row, dim, o[i].x * f, o[i].y * f);
        write_pair(c.seq, head0 + row, dim + 2, o[i].z * f, o[i].w * f);
      }
    }
  };
  // This warp has stored a piece of c's unit.  The last of the warps that do joins them, in the order of the
  // list: the sum does not depend on who that is.
  auto arrive = [&](const DenseCursor& c, const DensePieces& all) {
    __threadfence();
    __syncwarp();
    uint32_t* counter = p.counters + int64_t(all.first) * p.side + member;
    uint32_t seen = 0;
    if (lane == 0) seen = atomicAdd(counter, 1u);
    seen = __shfl_sync(0xffffffffu, seen, 0);
    if (seen + 1 != uint32_t(all.count)) return;
    __threadfence();
    if (lane == 0) *counter = 0u;
    join(std::false_type{}, c, all.count, [&](int i) {
      const int r = dense_piece_run(cut, all, i);
      return piece_of(r, dense_slot(cut, r, c.a));
    }, nullptr);
  };

  // ---- stream ------------------------------------------------------------------------------------------
  // (all teams of the CTA inside one unit group: they merge at the end)
  bool merging = false;
  if (teams > 1 && cut.begin(blockIdx.x * teams) < cut.total) {
    DenseCursor c;
    start(c, blockIdx.x * teams);
    merging = dense_cta_merges(cut, blockIdx.x, c.a, c.b);
  }
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue(i);
  int stage = 0;
  bool any_bad = false;
  bool begun_before = false;  // the run's first unit has left a piece
  DenseCursor before;
  for (bool first = true; cu.at < cu.end; first = false) {
    issue(stage == 0 ? S::kStages - 1 : stage - 1);
    if (first || cu.at == cu.a) begin_unit();
    cp_async_wait<S::kStages - 1>();
    __syncwarp();
    any_bad |= (bad >> stage) & 1;
    tile_step(stage);
    __syncwarp();
    if (cu.at + 1 == cu.end) break;
    if (cu.at + 1 == cu.b) {
      if (cu.a >= cut.begin(run)) {
        flush(nullptr);
      } else {  // the join, if it falls to this warp, needs the ring: at the end
        flush(piece_of(run, 0));
        begun_before = true;
        before = cu;
      }
    }
    advance(cu);
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
  }
  if (cut.begin(run) >= cut.end(run)) return;
  if (any_bad && lane == 0) atomicOr(p.status, FQ_DEV_BAD_BLOCK_INDEX);
  cp_async_wait<0>();
  __syncwarp();
  const bool whole = cu.a >= cut.begin(run) && cu.b <= cut.end(run);
  if (!merging) {
    if (whole) flush(nullptr); else flush(piece_of(run, dense_slot(cut, run, cu.a)));
    if (begun_before) arrive(before, dense_pieces(cut, before.a, before.b));
    if (!whole) arrive(cu, dense_pieces(cut, cu.a, cu.b));
    return;
  }
  flush(meet);
  __syncthreads();
  if (team > 0) return;
  const DensePieces all = dense_pieces(cut, cu.a, cu.b);
  float* dst = all.count == 1 ? nullptr : piece_of(run, dense_slot(cut, run, cu.a));
  join(std::true_type{}, cu, teams, [&](int i) {
    return reinterpret_cast<const float*>(smem + (i * p.side + warp) * S::kRing) + 33 * kRows;
  }, dst);
  if (dst) arrive(cu, all);
}

// ------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------
struct DenseGeometry {
  int chunks, rows, side, piece_floats;
  bool r16;
};
// Up to 8 query heads to a unit (16 where a KV head has more: its keys are then read half as often).
static DenseGeometry dense_geometry(int hq, int hkv, int d) {
  DenseGeometry x;
  const int group = hq / hkv;
  x.r16 = group > 8;
  x.chunks = (group + 15) / 16;
  x.rows = (group + x.chunks - 1) / x.chunks;
  const int warps = d > 128 ? 4 : 8;
  x.side = warps;  // adjacent units to the warps of a CTA, as many as divide a sequence's units
  while (hkv * x.chunks % x.side != 0) x.side /= 2;
  x.piece_floats = (x.rows * (d + 2) + 3) & ~3;
  return x;
}

// SMs of the current device; kernels whose shared memory has been asked for on it
struct DenseDevice {
  int device = -1, sms = 0;
};
static int dense_device(DenseDevice& known, bool& changed) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  changed = device != known.device;
  if (e == cudaSuccess && changed) {
    e = cudaDeviceGetAttribute(&known.sms, cudaDevAttrMultiProcessorCount, device);
    known.device = e == cudaSuccess ? device : -1;
  }
  return e == cudaSuccess ? FQ_OK : fail(FQ_ERR_CUDA, "dense decode: %s", cudaGetErrorString(e));
}
static int dense_sms(int& sms) {
  static thread_local DenseDevice known;
  bool changed;
  const int rc = dense_device(known, changed);
  sms = std::min(known.sms, kDenseMaxCtas);
  return rc;
}

template <typename T, int D, bool R16>
static int launch_dense(const DenseArgs& p, int ctas, cudaStream_t stream) {
  using S = DenseShape<D>;
  const size_t smem = S::kSmem + (2 * size_t(p.seqs) + 1) * sizeof(int);
  const auto kernel = dense_decode_kernel<T, D, R16>;
  static thread_local DenseDevice known;
  bool changed;
  if (const int rc = dense_device(known, changed)) return rc;
  if (changed) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               S::kSmem + (2 * kDenseMaxSeqs + 1) * int(sizeof(int)));
    if (e != cudaSuccess) {
      known.device = -1;
      return fail(FQ_ERR_CUDA, "dense decode: %s", cudaGetErrorString(e));
    }
  }
  kernel<<<ctas, S::kWarps * 32, smem, stream>>>(p);
  return check_launch("dense decode");
}
template <typename T, int D>
static int launch_dense(const DenseArgs& p, bool r16, int ctas, cudaStream_t stream) {
  return r16 ? launch_dense<T, D, true>(p, ctas, stream) : launch_dense<T, D, false>(p, ctas, stream);
}
template <typename T>
static int launch_dense(const DenseArgs& p, int d, bool r16, int ctas, cudaStream_t stream) {
  switch (d) {
    case 64: return launch_dense<T, 64>(p, r16, ctas, stream);
    case 96: return launch_dense<T, 96>(p, r16, ctas, stream);
    case 128: return launch_dense<T, 128>(p, r16, ctas, stream);
    default: return launch_dense<T, 256>(p, r16, ctas, stream);
  }
}

}  // namespace fq

using namespace fq;

static bool dense_shape_ok(int num_seqs, int hq, int hkv, int d) {
  return num_seqs >= 0 && num_seqs <= kDenseMaxSeqs && hkv > 0 && hq > 0 && hq % hkv == 0 && hq <= 1024 &&
         (d == 64 || d == 96 || d == 128 || d == 256);
}

extern "C" size_t fq_dense_paged_decode_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads,
                                                        int head_dim) {
  if (!dense_shape_ok(num_seqs, num_q_heads, num_kv_heads, head_dim)) return 0;
  const DenseGeometry x = dense_geometry(num_q_heads, num_kv_heads, head_dim);
  const size_t warps = head_dim > 128 ? 4 : 8;
  return kDenseHead + kDenseMaxCtas * warps * 2 * size_t(x.piece_floats) * sizeof(float);
}

extern "C" int fq_dense_paged_decode(
    const void* q, fq_dtype dtype, int64_t q_seq_stride, int64_t q_head_stride, const void* key_cache,
    int64_t k_block_stride, int64_t k_token_stride, int64_t k_head_stride, const void* value_cache,
    int64_t v_block_stride, int64_t v_token_stride, int64_t v_head_stride, const int32_t* block_table,
    int64_t block_table_stride, int block_table_width, const int32_t* seq_lens, int num_seqs, int num_q_heads,
    int num_kv_heads, int head_dim, int block_size, int64_t num_blocks, float sm_scale, int window, void* out,
    float* lse, void* workspace, size_t workspace_bytes, fq_stream_t stream) {
  FQ_RANGE("fq_dense_paged_decode");
  FQ_REQUIRE(num_seqs >= 0 && window >= 0 && block_table_width >= 0 && num_blocks >= 0, FQ_ERR_INVALID_ARGUMENT,
             "dense decode: negative size");
  FQ_REQUIRE(dtype == FQ_F16 || dtype == FQ_BF16, FQ_ERR_UNSUPPORTED, "dense decode: pages are fp16 or bf16");
  FQ_REQUIRE(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0, FQ_ERR_INVALID_ARGUMENT,
             "dense decode: %d query heads on %d KV heads", num_q_heads, num_kv_heads);
  FQ_REQUIRE(dense_shape_ok(num_seqs, num_q_heads, num_kv_heads, head_dim), FQ_ERR_UNSUPPORTED,
             "dense decode: head_dim 64, 96, 128 or 256, at most %d sequences and 1024 query heads (got %d, %d, %d)",
             kDenseMaxSeqs, head_dim, num_seqs, num_q_heads);
  FQ_REQUIRE(block_size > 0 && block_size % kDenseTile == 0, FQ_ERR_UNSUPPORTED,
             "dense decode: block_size must be a multiple of %d (got %d)", kDenseTile, block_size);
  if (num_seqs == 0) return FQ_OK;
  FQ_REQUIRE(q && seq_lens && out, FQ_ERR_INVALID_ARGUMENT, "dense decode: null pointer");
  FQ_REQUIRE(block_table_width == 0 || (block_table && key_cache && value_cache), FQ_ERR_INVALID_ARGUMENT,
             "dense decode: null pointer");
  FQ_REQUIRE(aligned(key_cache, 16) && aligned(value_cache, 16) && (k_block_stride | k_token_stride | k_head_stride |
             v_block_stride | v_token_stride | v_head_stride) % 8 == 0, FQ_ERR_ALIGNMENT,
             "dense decode: rows of the caches must start at multiples of 16 bytes");
  FQ_REQUIRE(aligned(q, 4) && (q_seq_stride | q_head_stride) % 2 == 0 && aligned(out, 4), FQ_ERR_ALIGNMENT,
             "dense decode: rows of q and out must start at multiples of 4 bytes");
  const DenseGeometry x = dense_geometry(num_q_heads, num_kv_heads, head_dim);
  const int64_t unit_groups = int64_t(num_kv_heads) * x.chunks / x.side;
  const int64_t most = num_seqs * unit_groups * block_table_width * (block_size / kDenseTile);
  FQ_REQUIRE(most < (int64_t(1) << 30), FQ_ERR_UNSUPPORTED, "dense decode: block table of 2^30 tiles or more");
  FQ_REQUIRE(workspace && aligned(workspace, 16) &&
                 workspace_bytes >= fq_dense_paged_decode_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim),
             FQ_ERR_WORKSPACE, "dense decode: workspace missing, misaligned or too small");
  DenseArgs p;
  p.q = q; p.k = key_cache; p.v = value_cache; p.out = out; p.lse = lse;
  p.table = block_table; p.lens = seq_lens;
  p.q_seq = q_seq_stride; p.q_head = q_head_stride;
  p.k_block = k_block_stride; p.k_token = k_token_stride; p.k_head = k_head_stride;
  p.v_block = v_block_stride; p.v_token = v_token_stride; p.v_head = v_head_stride;
  p.table_stride = block_table_stride; p.num_blocks = num_blocks;
  p.seqs = num_seqs; p.hq = num_q_heads; p.hkv = num_kv_heads;
  p.table_width = block_table_width; p.block_size = block_size; p.window = window;
  p.chunks = x.chunks; p.rows = x.rows; p.side = x.side; p.piece_floats = x.piece_floats;
  p.scale_log2 = sm_scale * 1.44269504f;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  p.status = reinterpret_cast<uint32_t*>(ws);
  p.counters = reinterpret_cast<uint32_t*>(ws + kDenseCounters);
  p.pieces = reinterpret_cast<float*>(ws + kDenseHead);
  // one CTA per SM (the rings fill its shared memory); no more than there can be runs, or rows without a token
  const int teams = (head_dim > 128 ? 4 : 8) / x.side;
  const int64_t runs = (most + kDenseShortest - 1) / kDenseShortest;
  const int64_t want = (runs + teams - 1) / teams;
  int sms = 0;
  if (const int rc = dense_sms(sms)) return rc;
  const int ctas = int(std::min<int64_t>(sms, std::max<int64_t>(want, std::min(num_seqs, 16))));
  return dtype == FQ_F16 ? launch_dense<__half>(p, head_dim, x.r16, ctas, stream)
                         : launch_dense<__nv_bfloat16>(p, head_dim, x.r16, ctas, stream);
}
