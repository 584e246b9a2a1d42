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
// out: dense_split.h.  Sixteen lanes find what the next sixteen tiles are and where they stand (the page's id on its
// way while earlier tiles are worked on) and leave that in shared memory.  Sums, maxima and weights are fp32; a
// weight enters the value product as two 16-bit terms (hi + lo, 2^-17 of it or better), so that the output is
// rounded once, at the end.  With up to eight query heads per unit the lo terms are the rows 8..15 of the A operand
// and cost nothing.
//
// What is left in pieces is joined by a second kernel, launched with the first (programmatic dependent launch).
// Joined in the first, by the last warp to arrive behind fences and a counter, 1 x 900 tokens took 20 us instead of 10,
// and one warp had to read all pieces of a long sequence.
//
// Measured (us the call, bytes of the keys and values a second): 32 x 4096, 32 / 8 heads of 128: 94, 5.7 TB/s; ragged
// 8 x 131072, 64 / 8: 433 - 445, 6.6; 48 windows of 1000, 16 / 16 heads of 64: 43, 4.6; 64 x 2000, 16 / 8 of 256: 166, 6.3; 1 x
// 900: 10.3 us, of which the first tile is computed at 5 and the join takes 3.
#include <algorithm>

#include <cooperative_groups.h>

#include "dense_split.h"
#include "fq_common.cuh"

namespace fq {

namespace cg = cooperative_groups;

constexpr int kDenseMaxCtas = 148;
constexpr int kDenseMaxSeqs = 2048;
// Workspace: the head (status word; the number of runs taken), zero between calls; the list's bounds of the
// sequences; pieces.
constexpr size_t kDenseTickets = 64, kDenseBounds = 32768, kDensePieces = kDenseBounds + 16384;
static_assert((kDenseMaxSeqs + 1) * sizeof(int) <= kDensePieces - kDenseBounds, "");

struct DenseArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int32_t *table, *lens;
  int64_t q_seq, q_head;                 // strides, in elements
  int64_t k_block, k_token, k_head, v_block, v_token, v_head;
  int64_t table_stride, num_blocks;
  int seqs, hq, hkv, table_width, block_size, window;
  int chunks, rows, group;               // units of a KV head, query heads of a unit and of a KV head
  int side_bits, unit_groups;            // units side by side (a power of two), such groups of a sequence
  int piece_floats;                      // stride of the pieces
  float scale_log2;
  int fixed;                             // runs dealt out beforehand
  int join_rows, join_wide, join_wides;  // heads and dimensions of a CTA of the join, such parts of a head
  int join_columns, join_groups;         // its columns of four dimensions, threads to each of them
  int join_split;                        // CTAs of its cluster
  uint32_t *status, *tickets;
  int* bounds;
  float* pieces;                         // [slot][side]: [rows][D], [rows][2] (maximum, sum)
};

// Warps of a CTA, one CTA per SM: as many as the registers leave (a row of the accumulators is D floats).  head_dim 64,
// 48 x 1000 tokens: 45 us with 8, 41 with 16.
__host__ __device__ constexpr int dense_warps(int d) { return d == 64 ? 16 : (d > 128 ? 4 : 8); }

template <int D, bool R16>
struct DenseShape {
  static constexpr int kWarps = dense_warps(D);
  static constexpr int kRow = 2 * D;         // bytes
  static constexpr int kTensor = kDenseTile * kRow;
  static constexpr int kStage = 2 * kTensor;
  static constexpr int kStages = D == 96 ? 4 : 3;  // 192 KB in all
  static constexpr int kRing = kStages * kStage;
  static constexpr int kDescribed = kWarps * 32 * 16;  // 32 tiles of a warp
  // An A operand is four registers in a row: with up to 8 query heads half of them are zeros, 64 registers in all at
  // head_dim 256, which spills (64 x 2000 tokens, 16 / 8 heads: 198 - 219 us).  There the queries stand in shared
  // memory, and a chunk of zeros for the other rows (166 us).
  static constexpr bool kQueries = D == 256 && !R16;
  static constexpr int kQuery = 8 * kRow;
  static constexpr int kZeros = kWarps * kRing + kDescribed + kWarps * kQuery;
  static constexpr int kSmem = kQueries ? kZeros + 16 : kWarps * kRing + kDescribed;
  // The 16-byte chunks of a row are permuted, so that the same chunk of 8 rows stands in all banks.
  static __device__ __forceinline__ int key(int row) { return D == 96 ? row >> 1 & 3 : row & 7; }
};

// (keys and values are read once: with a hint that keeps the L2 for what is used again, the pieces, the tables and
// the kernels' code among it)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0), "l"(policy)
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

// A tile: x the page (-1: none), y the first token in it | first visible row << 22 | row behind the last << 26,
// z sequence | unit << 12 | first of the unit << 30 | last << 31 (of what this run has of it), w the piece (-1: all
// of the unit is here).
constexpr int kDenseMaxBlock = 1 << 22;

struct DenseUnit {
  int head0, count;  // query heads
};
__device__ __forceinline__ DenseUnit dense_unit(const DenseArgs& p, int unit) {
  const int kv = p.chunks == 1 ? unit : unit / p.chunks, chunk = unit - kv * p.chunks;
  return {kv * p.group + chunk * p.rows, min(p.rows, p.group - chunk * p.rows)};
}
__device__ __forceinline__ float dense_lse(float m, float l, float lift) {
  return l == 0.f ? -INFINITY : (m + log2f(l) - lift) * 0.69314718f;
}

template <typename T, int D, bool R16>
__global__ void __launch_bounds__(DenseShape<D, R16>::kWarps * 32, 1) dense_decode_kernel(const DenseArgs p) {
  using S = DenseShape<D, R16>;
  using X = Dense16<T>;
  constexpr int kSteps = D / 16, kBlocks = D / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int warp_total[S::kWarps];
  __shared__ DenseCut cut;  // (ten registers less, where head_dim 256 has none to spare)
  int4* const described = reinterpret_cast<int4*>(smem + S::kWarps * S::kRing);
  int* const prefix = reinterpret_cast<int*>(smem + S::kSmem);  // [seqs + 1]
  int* const lengths = prefix + p.seqs + 1;                     // [seqs]
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int g = lane >> 2, t = lane & 3;
  const int64_t room = int64_t(p.table_width) * p.block_size;
  const int unit_groups = p.unit_groups;
  if (S::kQueries && tid < 4) reinterpret_cast<uint32_t*>(smem + S::kZeros)[tid] = 0u;
  // (the wait first: the second kernel, which this lets start, reads what the kernels before this one have written)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

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
    for (int s = s0; s < s1; ++s) {
      prefix[s + 1] += before;
      if (blockIdx.x == 0) p.bounds[s + 1] = prefix[s + 1];
    }
    if (blockIdx.x == 0 && tid == 0) p.bounds[0] = 0;
    if (tid == S::kWarps * 32 - 1) cut = dense_cut(before + sum, p.fixed, p.seqs * unit_groups);
    __syncthreads();
  }
  const int groups_all = p.seqs * unit_groups;

  // ---- the warp's tiles, described sixteen at a time ---------------------------------------------------
  const int tiles_per_block = p.block_size / kDenseTile;
  const uint32_t taken = uint32_t(cut.taken()) << p.side_bits;
  int4* const mine = described + warp * 32;
  const int here = blockIdx.x * S::kWarps + warp;
  int run = here >> p.side_bits, member = here - (run << p.side_bits);
  int at = cut.begin(run), end = cut.end(run);
  uint32_t ticket = 0;  // (lane 0) the next run, where it has been asked for
  bool asked = false;
  auto ask = [&] {
    if (taken && lane == 0) ticket = atomicAdd(p.tickets, 1u);
    asked = true;
  };
  int made = 0, issued = 0, used = 0;  // tiles described, on their way, done
  int waiting = 0;                     // described in `next`, not stored yet
  bool finished = false;
  int4 next;
  auto describe = [&] {
    if (at == end) {
      if (!asked) ask();
      asked = false;
      const uint32_t x = __shfl_sync(0xffffffffu, ticket, 0);
      if (x >= taken) {
        // (every warp gets one that is too large: the last of them leaves the counter as it was found)
        if (taken && lane == 0 && x == taken + gridDim.x * S::kWarps - 1) *p.tickets = 0u;
        finished = true;
        return;
      }
      run = cut.fixed + int(x >> p.side_bits);
      member = x & ((1 << p.side_bits) - 1);
      at = cut.begin(run);
      end = cut.end(run);
    }
    waiting = min(16, end - at);
    if (lane < waiting) {
      const bool tail = cut.is_tail(run);
      const int i = at + lane, here = cut.entry(tail, i);
      int lo = 0, hi = p.seqs - 1;  // the sequence whose entries hold `here`
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid + 1] > here) hi = mid; else lo = mid + 1;
      }
      const DenseSpan span = dense_span(lengths[lo], room, p.window);
      const int group = unit_groups == 1 ? 0 : (here - prefix[lo]) / span.tiles;
      const int a = prefix[lo] + group * span.tiles, b = a + span.tiles;
      const int tile = span.first_tile + here - a;
      const int page = tile / tiles_per_block, first = tile * kDenseTile;
      next.x = __ldg(p.table + lo * p.table_stride + page);
      next.y = (tile - page * tiles_per_block) * kDenseTile | max(span.begin - first, 0) << 22 |
               min(span.len - first, kDenseTile) << 26;
      next.z = lo | ((group << p.side_bits) + member) << 12;
      if (i == cut.kind_of(tail, a) || i == cut.begin(run)) next.z |= 1 << 30;
      if (i + 1 == cut.kind_of(tail, b) || i + 1 == end) next.z |= 1 << 31;
      const int nth = lo * unit_groups + group;
      next.w = dense_whole(cut, run, a, b) ? -1 : (dense_slot(cut, run, nth, groups_all, a) << p.side_bits) + member;
    }
    at += waiting;
  };
  auto store = [&] {
    if (lane < waiting) {
      if (unsigned(next.x) >= uint64_t(p.num_blocks)) {
        next.x = -1;
        atomicOr(p.status, FQ_DEV_BAD_BLOCK_INDEX);
      }
      mine[(made + lane) & 31] = next;
    }
    made += waiting;
    waiting = 0;
    __syncwarp();
  };

  const uint32_t ring = smem_u32(smem) + warp * S::kRing;
  const uint64_t policy = l2_evict_first_policy();
  constexpr int kPerRow = D / 8, kChunks = kDenseTile * kPerRow / 32;
  // one tile on its way, if there is one (each call is a group: tile n is complete when group n is)
  auto issue = [&](int stage) {
    while (issued == made && !finished) {
      if (!waiting) describe();
      store();
    }
    if (issued < made) {
      const int4 d = mine[issued & 31];
      ++issued;
      const int unit = (d.z >> 12) & 0x3fff, head = p.chunks == 1 ? unit : unit / p.chunks;
      const int row = d.y & (kDenseMaxBlock - 1);
      const int64_t id = d.x < 0 ? 0 : d.x;
      const T* k = static_cast<const T*>(p.k) + id * p.k_block + row * p.k_token + head * p.k_head;
      const T* v = static_cast<const T*>(p.v) + id * p.v_block + row * p.v_token + head * p.v_head;
      const int lo = (d.y >> 22) & 15, hi = d.x < 0 ? 0 : (d.y >> 26) & 31;
      const uint32_t dst = ring + stage * S::kStage;
      // (the rows of a tile stand in one page: those outside the sequence have an address, and nothing is read there)
      const int r0 = lane / kPerRow, col = lane % kPerRow;
      const T *ks = k + r0 * p.k_token + col * 8, *vs = v + r0 * p.v_token + col * 8;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if constexpr (32 % kPerRow == 0) {
          constexpr int kRows = 32 / kPerRow;
          const int r = r0 + c * kRows;
          const bool valid = r >= lo && r < hi;
          const uint32_t to = dst + r * S::kRow + ((col ^ S::key(r)) << 4);
          cp_async16(to, ks, valid, policy);
          cp_async16(to + S::kTensor, vs, valid, policy);
          ks += kRows * p.k_token;
          vs += kRows * p.v_token;
        } else {
          const int i = lane + 32 * c, r = i / kPerRow, at = i % kPerRow;
          const bool valid = r >= lo && r < hi;
          const uint32_t to = dst + r * S::kRow + ((at ^ S::key(r)) << 4);
          cp_async16(to, k + r * p.k_token + at * 8, valid, policy);
          cp_async16(to + S::kTensor, v + r * p.v_token + at * 8, valid, policy);
        }
      }
    }
    cp_async_commit();
  };

  // ---- state of the unit in work ----------------------------------------------------------------------
  uint32_t qf[S::kQueries ? 1 : kSteps][R16 ? 4 : 2];
  unsigned char* const queries = smem + S::kWarps * S::kRing + S::kDescribed + warp * S::kQuery;  // (kQueries)
  float acc[kBlocks][4];
  float top[R16 ? 2 : 1], sum[R16 ? 2 : 1];

  auto begin_unit = [&](const int4& d) {
    const DenseUnit u = dense_unit(p, (d.z >> 12) & 0x3fff);
    const T* q = static_cast<const T*>(p.q) + (d.z & 0xfff) * p.q_seq + u.head0 * p.q_head;
    if constexpr (S::kQueries) {
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const int word = lane + 32 * i;  // of the row
          const uint32_t x = r < u.count ? *reinterpret_cast<const uint32_t*>(q + r * p.q_head + 2 * word) : 0u;
          *reinterpret_cast<uint32_t*>(queries + r * S::kRow + ((word / 4 ^ S::key(r)) << 4) + word % 4 * 4) = x;
        }
    }
#pragma unroll
    for (int r = 0; r < (R16 ? 2 : 1); ++r) {
      const bool real = g + 8 * r < u.count;
      const T* row = q + (real ? (g + 8 * r) * p.q_head : 0) + 2 * t;
#pragma unroll
      for (int s = 0; s < (S::kQueries ? 0 : kSteps); ++s) {
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

  auto tile_step = [&](int stage, const int4& d) {
    const uint32_t kt = ring + stage * S::kStage, vt = kt + S::kTensor;
    const int mid = lane >> 3;
    // scores: rows = heads, columns = tokens (two blocks of eight)
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    const int k_row = (mid >> 1) * 8 + (lane & 7), v_row = (mid & 1) * 8 + (lane & 7);
    // (kQueries) rows 0 - 7 for the lanes of the first and third matrix, zeros for the others
    const uint32_t q_real = ~mid & 1, q_key = ((mid >> 1) ^ S::key(lane & 7)) << 4;
    const uint32_t qa = q_real ? smem_u32(queries) + (lane & 7) * S::kRow : smem_u32(smem + S::kZeros);
    const uint32_t ka = kt + k_row * S::kRow, k_key = ((mid & 1) ^ S::key(k_row)) << 4;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      uint32_t b[4];
      ldmatrix4(b, ka + (i * 32 ^ k_key));
      uint32_t a[4];
      if constexpr (S::kQueries) {
        ldmatrix4(a, qa + (i * 32 ^ q_key) * q_real);
      } else if constexpr (R16) {
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
    const int lo = (d.y >> 22) & 15, hi = d.x < 0 ? 0 : (d.y >> 26) & 31;
    if (lo > 0 || hi < kDenseTile) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = n * 8 + 2 * t + (e & 1);
          if (at < lo || at >= hi) s[n][e] = -INFINITY;
        }
    }
    uint32_t hi_a[4];
    [[maybe_unused]] uint32_t lo_a[4];
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
    const uint32_t va = vt + v_row * S::kRow, v_key = ((mid >> 1) ^ S::key(v_row)) << 4;
#pragma unroll
    for (int j = 0; j < kBlocks; j += 2) {
      uint32_t b[4];
      ldmatrix4_trans(b, va + (j * 16 ^ v_key));
      X::mma(acc[j], hi_a, b[0], b[1]);
      X::mma(acc[j + 1], hi_a, b[2], b[3]);
      if constexpr (R16) {
        X::mma(acc[j], lo_a, b[0], b[1]);
        X::mma(acc[j + 1], lo_a, b[2], b[3]);
      }
    }
  };

  // the unit, or what the run has of it: to `out`, or as a piece
  auto flush = [&](const int4& d) {
    const int seq = d.z & 0xfff;
    const DenseUnit u = dense_unit(p, (d.z >> 12) & 0x3fff);
    float* const dst = p.pieces + int64_t(d.w) * p.piece_floats;
#pragma unroll
    for (int r = 0; r < (R16 ? 2 : 1); ++r) {
      float l = sum[r];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const int row = g + 8 * r;
      if (row >= u.count) continue;
      const int64_t out_row = int64_t(seq) * p.hq + u.head0 + row;
      const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        float x = acc[j][2 * r], y = acc[j][2 * r + 1];
        if constexpr (!R16) {  // the lo terms
          x += acc[j][2];
          y += acc[j][3];
        }
        if (d.w >= 0)
          *reinterpret_cast<float2*>(dst + row * D + 8 * j + 2 * t) = make_float2(x, y);
        else
          *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + out_row * D + 8 * j + 2 * t) = X::pack(x * f, y * f);
      }
      if (t == 0) {
        if (d.w >= 0)
          *reinterpret_cast<float2*>(dst + p.rows * D + 2 * row) = make_float2(top[r], l);
        else if (p.lse)
          p.lse[out_row] = dense_lse(top[r], l, X::kLift);
      }
    }
  };

  // ---- stream ------------------------------------------------------------------------------------------
  int into = 0, from = 0;  // stages
#pragma unroll 1
  for (int step = 0;; ++step) {
    // The next tiles are described when eight are left, and stored, with their pages' ids, when four are.  A run is taken
    // no sooner than its first tile can follow the last one: one that is held back is one that no other warp takes.
    if (waiting) {
      if (made - issued <= 4) store();
    } else if (!finished && made - issued <= 8) {
      if (at < end || made - issued <= 1) describe();
      else if (!asked && made - issued <= 2) ask();
    }
    issue(into);
    into = into + 1 == S::kStages ? 0 : into + 1;
    if (step < S::kStages - 1) continue;
    if (used == made) break;
    const int4 d = mine[used & 31];
    if (d.z & 1 << 30) begin_unit(d);
    cp_async_wait<S::kStages - 1>();
    __syncwarp();
    tile_step(from, d);
    if (d.z < 0) flush(d);
    __syncwarp();
    ++used;
    from = from + 1 == S::kStages ? 0 : from + 1;
  }
  cp_async_wait<0>();
}

// A cluster for `join_rows` query heads of a unit, or of a few units one after the other, and `join_wide` of their
// dimensions, each of its CTAs for a part of the pieces: their weights first, a warp to a head and a lane to a piece, then
// the sums, a group of threads to a piece, and the first CTA adds up what the others have in their shared memory.  A unit
// that one run had is left alone; heads without tokens get zeros.  The first pieces are on their way with the weights.
constexpr int kJoinThreads = 128, kJoinPieces = 128, kJoinRows = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads, 8) dense_join_kernel(const DenseArgs p) {
  constexpr int kAhead = 4;
  __shared__ float weights[kJoinRows][kJoinPieces];
  __shared__ float totals[kJoinRows][3];  // maximum, sum, factor of what stands
  __shared__ float4 sums[kJoinThreads];
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int unit_groups = p.unit_groups, units = unit_groups << p.side_bits, seq = blockIdx.z / p.join_split;
  const unsigned part = blockIdx.z - seq * p.join_split, parts = p.join_split;  // of the pieces
  const int row0 = blockIdx.y / p.join_wides * p.join_rows, wide = blockIdx.y % p.join_wides;
  const int columns = p.join_columns, groups = p.join_groups;
  const int mine = tid / columns, column = tid - mine * columns;
  const int row = column * 4 / p.join_wide;
  const int dim = wide * p.join_wide + column * 4 - row * p.join_wide;
  // Nothing that another kernel has written is read before this wait, the lengths neither: the first kernel has waited for
  // what came before it, but what a kernel sees is promised behind a wait of its own only (1 x 900 tokens: 9.5 us with the
  // lengths read before it).  No CTA leaves before it: this kernel must not end before the first one has.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int s0 = p.bounds[seq], tiles = (p.bounds[seq + 1] - s0) / unit_groups, total = p.bounds[p.seqs];
  const bool with_lse = p.lse && wide == 0 && part == 0;
  const int groups_all = p.seqs * unit_groups;
  const DenseCut cut = dense_cut(total, p.fixed, groups_all);
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int group = unit >> p.side_bits, member = unit - (group << p.side_bits);
    const DenseUnit u = dense_unit(p, unit);
    const int rows = min(p.join_rows, u.count - row0);
    const bool real = row < rows && mine < groups;
    const int64_t out_row = int64_t(seq) * p.hq + u.head0 + row0;
    auto write = [&](float4 o) {
      uint2 x;
      x.x = Dense16<T>::pack(o.x, o.y);
      x.y = Dense16<T>::pack(o.z, o.w);
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (out_row + row) * D + dim) = x;
    };
    const int a = s0 + group * tiles;
    const DensePieces all = dense_pieces(cut, a, a + tiles);
    const int pieces = all.count(), first = pieces * part / parts, n = pieces * (part + 1) / parts;
    if (tiles == 0 && part == 0) {
      if (real && mine == 0) write(make_float4(0.f, 0.f, 0.f, 0.f));
      if (with_lse && tid < rows) p.lse[out_row + tid] = -INFINITY;
    }
    if (tiles == 0 || pieces == 1 || rows <= 0) continue;
    __syncthreads();  // what the unit before had in shared memory has been read
    const int nth = seq * unit_groups + group;
    auto piece = [&](int i) {
      return p.pieces + ((int64_t(dense_slot(cut, all.run(i), nth, groups_all, a)) << p.side_bits) + member) * p.piece_floats;
    };
    const int64_t offset = (row0 + row) * D + dim;
    float m = -INFINITY, l = 0.f;  // of row `warp`
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float w, const float4& v) {
      o.x = fmaf(w, v.x, o.x);
      o.y = fmaf(w, v.y, o.y);
      o.z = fmaf(w, v.z, o.z);
      o.w = fmaf(w, v.w, o.w);
    };
    if (tid < kJoinRows) {
      totals[tid][0] = -INFINITY;
      totals[tid][1] = 0.f;
    }
    for (int i0 = first; i0 < n; i0 += kJoinPieces) {
      const int some = min(kJoinPieces, n - i0);
      float4 ahead[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = mine + k * groups;
        if (real && i < some) ahead[k] = *reinterpret_cast<const float4*>(piece(i0 + i) + offset);
      }
      __syncthreads();  // the weights before have been used
      if (warp < rows) {
        float2 x[kJoinPieces / 32];
        float now = m;
#pragma unroll
        for (int k = 0; k < kJoinPieces / 32; ++k) {
          const int i = lane + 32 * k;
          x[k] = make_float2(-INFINITY, 0.f);
          if (i < some) x[k] = *reinterpret_cast<const float2*>(piece(i0 + i) + p.rows * D + 2 * (row0 + warp));
        }
#pragma unroll
        for (int k = 0; k < kJoinPieces / 32; ++k) now = fmaxf(now, x[k].x);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, s));
        const float ref = now == -INFINITY ? 0.f : now, f = fast_exp2(m - ref);
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < kJoinPieces / 32; ++k) {
          const float w = fast_exp2(x[k].x - ref);
          s = fmaf(w, x[k].y, s);
          weights[warp][lane + 32 * k] = w;
        }
        l = fmaf(l, f, warp_sum(s));
        m = now;
        if (lane == 0) {
          totals[warp][0] = m;
          totals[warp][1] = l;
          totals[warp][2] = f;
        }
      }
      __syncthreads();
      if (!real) continue;
      const float f = totals[row][2];
      o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = mine + k * groups;
        if (i < some) add(weights[row][i], ahead[k]);
      }
#pragma unroll 6
      for (int i = mine + kAhead * groups; i < some; i += groups)
        add(weights[row][i], *reinterpret_cast<const float4*>(piece(i0 + i) + offset));
    }
    sums[tid] = o;
    __syncthreads();
    if (real && mine == 0) {
      for (int i = 1; i < groups; ++i) add(1.f, sums[i * columns + column]);
      sums[tid] = o;
    }
    if (parts > 1) cluster_barrier();
    if (part == 0) {
      float top = -INFINITY, sum = 0.f;  // of all CTAs, of the thread's row
      if (real && mine == 0) {
        for (unsigned z = 0; z < parts; ++z) top = fmaxf(top, cluster.map_shared_rank(&totals[row][0], z)[0]);
        const float ref = top == -INFINITY ? 0.f : top;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (unsigned z = 0; z < parts; ++z) {
          const float* of = cluster.map_shared_rank(&totals[row][0], z);
          const float w = fast_exp2(of[0] - ref);
          sum = fmaf(w, of[1], sum);
          add(w, *cluster.map_shared_rank(&sums[tid], z));
        }
        const float f = sum == 0.f ? 0.f : 1.f / sum;
        write(make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
        if (with_lse && column * 4 == row * p.join_wide) p.lse[out_row + row] = dense_lse(top, sum, Dense16<T>::kLift);
      }
    }
    if (parts > 1) cluster_barrier();  // what the first CTA reads stays
  }
}

// ------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------
struct DenseGeometry {
  int chunks, rows, group, side_bits, piece_floats;
  bool r16;
};
// Up to 8 query heads to a unit, 16 where a KV head has more: its keys are then read half as often (64 x 4000 tokens, 20 / 2
// heads: 71 us with units of 8, 56 with 16; 32 / 2: 72, 57).
static DenseGeometry dense_geometry(int hq, int hkv, int d) {
  DenseGeometry x;
  x.group = hq / hkv;
  x.r16 = x.group > 8;
  x.chunks = (x.group + 15) / 16;
  x.rows = (x.group + x.chunks - 1) / x.chunks;
  x.side_bits = 0;  // adjacent units to the warps of a CTA, as many as divide a sequence's units
  while (2 << x.side_bits <= dense_warps(d) && hkv * x.chunks % (2 << x.side_bits) == 0) ++x.side_bits;
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

// Programmatic dependent launch: the kernel's CTAs may start while the one before it on the stream ends, and wait for it
// themselves.
static int launch_dependent(void (*kernel)(DenseArgs), const DenseArgs& p, dim3 grid, int threads, size_t smem,
                            int cluster, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;  // the CTAs along z
  attributes[1].val.clusterDim.x = attributes[1].val.clusterDim.y = 1;
  attributes[1].val.clusterDim.z = cluster;
  config.attrs = attributes;
  config.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, p);
  if (e != cudaSuccess) return fail(FQ_ERR_CUDA, "dense decode: %s", cudaGetErrorString(e));
  return check_launch("dense decode");
}

// As few heads to a CTA of the join as leave it with eight CTAs on an SM, all resident at once.  Where that leaves room, the
// pieces of a unit are split over a cluster, 64 or fewer to a CTA (1 x 131072 tokens, 8 query heads on one KV head: 47 us the
// call without, 27 with), and the dimensions of a head where it still has more than 24 (1 x 900: 13.9 us with whole
// heads, 10.3 with 32 dimensions; 1 x 32768: 33.6 whichever is split first).
template <typename T, int D>
static int launch_join(DenseArgs p, cudaStream_t stream) {
  const int64_t units = int64_t(p.seqs) * p.hkv * p.chunks, most = 8 * kDenseMaxCtas;
  const int64_t tiles = int64_t(p.table_width) * (p.block_size / kDenseTile);
  const int64_t pieces = std::min(tiles, (int64_t(p.fixed) << p.side_bits) / units + 1);  // of a unit, about
  p.join_rows = 1;
  p.join_wide = D;
  p.join_split = 1;
  const auto ctas = [&] {
    return units * ((p.rows + p.join_rows - 1) / p.join_rows) * (D / p.join_wide) * p.join_split;
  };
  while (p.join_rows < p.rows && 2 * p.join_rows <= kJoinRows && 2 * p.join_rows * p.join_wide / 4 <= kJoinThreads &&
         ctas() > most)
    p.join_rows *= 2;
  while (p.join_split < 8 && pieces > 64 * p.join_split && 2 * ctas() <= most) p.join_split *= 2;
  if (pieces > 24 * p.join_split) {
    if (ctas() * (D / 32) <= most) p.join_wide = 32;
    else if (D % 64 == 0 && ctas() * (D / 64) <= most) p.join_wide = 64;
  }
  p.join_wides = D / p.join_wide;
  p.join_columns = p.join_rows * p.join_wide / 4;
  p.join_groups = kJoinThreads / p.join_columns;
  const int64_t over = (ctas() + most - 1) / most;  // units of a sequence that a CTA takes (1 where there is a split)
  const dim3 grid(unsigned((p.hkv * p.chunks + over - 1) / over),
                  (p.rows + p.join_rows - 1) / p.join_rows * p.join_wides, p.seqs * p.join_split);
  return launch_dependent(dense_join_kernel<T, D>, p, grid, kJoinThreads, 0, p.join_split, stream);
}

template <typename T, int D, bool R16>
static int launch_dense(const DenseArgs& p, int ctas, cudaStream_t stream) {
  using S = DenseShape<D, R16>;
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
  if (const int rc = launch_dependent(kernel, p, dim3(ctas), S::kWarps * 32, smem, 1, stream)) return rc;
  return launch_join<T, D>(p, stream);
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
  const int teams = dense_warps(head_dim) >> x.side_bits;
  return kDensePieces + (size_t(dense_slots(kDenseMaxCtas * teams)) << x.side_bits) * x.piece_floats * sizeof(float);
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
  FQ_REQUIRE(block_size > 0 && block_size % kDenseTile == 0 && block_size <= kDenseMaxBlock, FQ_ERR_UNSUPPORTED,
             "dense decode: block_size must be a multiple of %d, at most 2^22 (got %d)", kDenseTile, block_size);
  if (num_seqs == 0) return FQ_OK;
  FQ_REQUIRE(q && seq_lens && out, FQ_ERR_INVALID_ARGUMENT, "dense decode: null pointer");
  FQ_REQUIRE(block_table_width == 0 || (block_table && key_cache && value_cache), FQ_ERR_INVALID_ARGUMENT,
             "dense decode: null pointer");
  FQ_REQUIRE(aligned(key_cache, 16) && aligned(value_cache, 16) && (k_block_stride | k_token_stride | k_head_stride |
             v_block_stride | v_token_stride | v_head_stride) % 8 == 0, FQ_ERR_ALIGNMENT,
             "dense decode: rows of the caches must start at multiples of 16 bytes");
  FQ_REQUIRE(aligned(q, 4) && (q_seq_stride | q_head_stride) % 2 == 0 && aligned(out, 8), FQ_ERR_ALIGNMENT,
             "dense decode: rows of q must start at multiples of 4 bytes, out at one of 8");
  const DenseGeometry x = dense_geometry(num_q_heads, num_kv_heads, head_dim);
  const int64_t unit_groups = int64_t(num_kv_heads) * x.chunks >> x.side_bits;
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
  p.chunks = x.chunks; p.rows = x.rows; p.group = x.group; p.side_bits = x.side_bits;
  p.unit_groups = int(unit_groups); p.piece_floats = x.piece_floats;
  p.scale_log2 = sm_scale * 1.44269504f;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  p.status = reinterpret_cast<uint32_t*>(ws);
  p.tickets = reinterpret_cast<uint32_t*>(ws + kDenseTickets);
  p.bounds = reinterpret_cast<int*>(ws + kDenseBounds);
  p.pieces = reinterpret_cast<float*>(ws + kDensePieces);
  // one CTA per SM (the rings fill its shared memory), no more than there can be runs
  int sms = 0;
  if (const int rc = dense_sms(sms)) return rc;
  const int teams = dense_warps(head_dim) >> x.side_bits;
  const int64_t runs = (most + kDenseShortest - 1) / kDenseShortest;
  const int ctas = int(std::max<int64_t>(1, std::min<int64_t>(sms, (runs + teams - 1) / teams)));
  p.fixed = ctas * teams;
  std::lock_guard<std::mutex> enqueued(workspace_calls(workspace));
  return dtype == FQ_F16 ? launch_dense<__half>(p, head_dim, x.r16, ctas, stream)
                         : launch_dense<__nv_bfloat16>(p, head_dim, x.r16, ctas, stream);
}
