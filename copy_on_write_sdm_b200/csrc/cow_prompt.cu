// cow_prompt.cu -- causal attention over packed prompts of different lengths, grouped heads.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale * q_i . k_j - m_i),   j <= i in i's own sequence
//
// A tile is some rows of one key head: neighbouring tokens times the key head's query heads, row =
// token * group + head, so that a group shares every key it reads and short prompts still fill
// their rows.  Keys pass in tiles; maximum, sum and output of the running softmax stay on the SM.
// Tiles run in the order of their work, longest first, over all sequences
// together: the tile at place l of its sequence reads l + 1 tiles' keys, so the tiles of place l
// are one for each sequence that has more than l, and one is found by a search
// over l with no table to build.

#include <cuda.h>

#include "cow_common.cuh"

namespace {

constexpr int kMaxGroup = 64;

struct PromptLaunch {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* starts;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  int32_t* status;  // may be null
  int32_t sequences, tokens, heads, kv_heads, group, width, dtype;
  float scale_log2;  // scale * log2(e)
};

// Sequence b as [begin, begin + count), inside the packed tokens whatever `starts` holds.
__device__ __forceinline__ int2 sequence_of(const PromptLaunch& P, int b) {
  const int begin = min(max(P.starts[b], 0), P.tokens), end = min(max(P.starts[b + 1], begin), P.tokens);
  return make_int2(begin, end - begin);
}

// The lane of the (n + 1)-th set bit of `has` (the same in the whole warp, n below its bits' number).
__device__ __forceinline__ int nth_lane(unsigned has, int n) {
  const int lane = threadIdx.x & 31;
  return __ffs(__ballot_sync(kFull, (has >> lane & 1) && __popc(has & ((1u << lane) - 1)) == n)) - 1;
}

struct Tile {
  int begin, count, first;  // its sequence, and its first token in it; count 0: none left
};

// Finds tiles by their place in the order of work; all members are one warp's.  A lane keeps the tile
// counts of kHeld sequences; those beyond 32 * kHeld are read again at every look.
struct TileFinder {
  static constexpr int kHeld = 4;
  int2 seq[kHeld];
  int held[kHeld];
  int most, all;

  __device__ __forceinline__ int tiles_of(const PromptLaunch& P, int tile_tokens, int b) const {
    return b < P.sequences ? (sequence_of(P, b).y + tile_tokens - 1) / tile_tokens : 0;
  }
  // tiles whose place in their sequence is >= h
  __device__ __forceinline__ int above(const PromptLaunch& P, int tile_tokens, int h) const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) n += max(held[i] - h, 0);
    for (int b = 32 * kHeld + (threadIdx.x & 31); b < P.sequences; b += 32) n += max(tiles_of(P, tile_tokens, b) - h, 0);
    return __reduce_add_sync(kFull, n);
  }
  __device__ __forceinline__ void begin(const PromptLaunch& P, int tile_tokens) {
    const int lane = threadIdx.x & 31;
    most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) seq[i] = 32 * i + lane < P.sequences ? sequence_of(P, 32 * i + lane) : make_int2(0, 0);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      held[i] = (seq[i].y + tile_tokens - 1) / tile_tokens;
      most = max(most, held[i]);
    }
    for (int b = 32 * kHeld + lane; b < P.sequences; b += 32) most = max(most, tiles_of(P, tile_tokens, b));
    most = __reduce_max_sync(kFull, most);
    all = above(P, tile_tokens, 0);
  }
  // The x-th tile in the order of work; none (count 0) from `all` on.
  __device__ __forceinline__ Tile find(const PromptLaunch& P, int tile_tokens, int x) const {
    const int lane = threadIdx.x & 31;
    Tile t{0, 0, 0};
    if (x >= all) return t;
    int lo = 0, hi = most;  // above(lo) > x >= above(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (above(P, tile_tokens, mid) > x) lo = mid; else hi = mid;
    }
    int rank = x - above(P, tile_tokens, hi);  // among the sequences with more than lo tiles
    t.first = lo * tile_tokens;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const unsigned has = __ballot_sync(kFull, held[i] > lo);
      if (rank >= 0 && rank < __popc(has)) {
        const int from = nth_lane(has, rank);
        t.begin = __shfl_sync(kFull, seq[i].x, from);
        t.count = __shfl_sync(kFull, seq[i].y, from);
      }
      rank -= __popc(has);
    }
    for (int base = 32 * kHeld; rank >= 0 && base < P.sequences; base += 32) {
      const unsigned has = __ballot_sync(kFull, tiles_of(P, tile_tokens, base + lane) > lo);
      if (rank < __popc(has)) {
        const int2 found = sequence_of(P, base + nth_lane(has, rank));
        t.begin = found.x;
        t.count = found.y;
      }
      rank -= __popc(has);
    }
    return t;
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// --------------------------------------------------------------------------
// f32
// --------------------------------------------------------------------------
//
// Every operand is held as three bf16 parts of eight bits each, which keep f32's exponent: no scale is shared, and nothing
// of one token, width or tile touches another's bits.  Six of the nine part products run on the bf16 matrix
// instructions with f32 sums, the other three being below f32's rounding: f32's accuracy at a sixth of the 16-bit rate.
// A tile of 64 keys is split once for the whole block.  Weights are 2^-8 at most, so that a sum of 256 of the
// type's largest values does not overflow before its division; products below 2^-126 are lost to the matrix
// instructions, so that values keep all 24 bits down to 2^-102 (2e-31).
// Values that are not finite are left out of the products (a weight of 0 times them is NaN) and added at
// the end to the rows that see them.
// Measured: sixteen prompts of 256, four heads of 32: 16.4 us back to back (31 us with the f32 pipe); 16 x 1,024 tokens,
// 32/8 heads of 128: 2.50 ms, 55 TFLOP/s of f32 work (330 of bf16 products, of about 560 that `mma.sync` gives here:
// 1,024 multiply-adds a cycle and SM); error against 64 bits 0.5 to 0.8 of plain f32 sums'.  (Two f16 parts under scales
// shared by a tile took 1.54 ms and were wrong wherever tokens of a tile lie far apart, those a row does not see among them.)
// Bound: the matrix instructions, 60 % of their rate, and the chain of split, scores, softmax and products of a key
// tile, with two or three warps to a scheduler.  Tried and not kept: all products of 16 widths in one go (2.43 ms, but
// cut off 24 or 48 times instead of 4 or 8: four times the error for heads of 128); of the form with f16 parts: two split
// tiles in turn with the next split beside the products, eight sums in turn instead of four (no change), tiles of 32 keys
// (12 % slower), four warps twice an SM (30 %), 128 keys for width 32.

constexpr int kKeys = 64;

template <int D>
struct F32Shape {
  static constexpr int kWarps = D > 64 ? 8 : 4;  // 16 rows each
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kRows = 16 * kWarps;
  static constexpr int kStride = D + 8;          // halves of a row in shared memory: rows apart by an odd number of 16 bytes
  static constexpr int kVecs = kKeys * D / 4 / kThreads;  // 16-byte words of a tile per thread
  static constexpr int kBytes = 2 * 3 * (kRows + 2 * kKeys) * kStride;
};

constexpr float kLeast = 1.1754943508222875e-38f;  // 2^-126
constexpr float kHeadroom = 8.f;                   // log2 of what weights lie below 1
__device__ __forceinline__ unsigned pack_bf162(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
// pairs of floats in one 64-bit register
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(uint64_t r) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(r));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// x in three bf16 parts of eight bits each, 24 together, which keep f32's exponent: the first is x cut off (a rounded
// one could overflow), the others are rounded.  Of what is not finite the second and third are NaN.
__device__ __forceinline__ uint3 split3(uint64_t x) {
  float2 f = both(x);
  uint3 p;
  p.x = __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x7632);
  x = fma2(pair(__uint_as_float(p.x << 16), __uint_as_float(p.x & 0xffff0000u)), pair(-1.f, -1.f), x);
  f = both(x);
  p.y = pack_bf162(f.x, f.y);
  f = both(fma2(pair(__uint_as_float(p.y << 16), __uint_as_float(p.y & 0xffff0000u)), pair(-1.f, -1.f), x));
  p.z = pack_bf162(f.x, f.y);
  return p;
}
__device__ __forceinline__ void mma_bf16(float* c, const unsigned* a, unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load_matrices(unsigned* r, const uint16_t* at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(at))
               : "memory");
}
__device__ __forceinline__ void load_matrices_turned(unsigned* r, const uint16_t* at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(at))
               : "memory");
}

constexpr int kBadWords = 8;  // 256 spans of key tiles

// Adds to a row's output the values of tokens up to `last` that are not finite, at two of every eight widths from `from` on.
// They lie in the spans of `per` key tiles that `bad` names, so that few of them cost little however long the prompt is.
__device__ __noinline__ void add_nonfinite_f32(const float* v, int64_t v_token, const unsigned* bad, int per, int last, float* out, int from,
                                               int width) {
  constexpr int kAtOnce = 16;
  for (int word = 0; word < kBadWords; ++word) {
    for (unsigned spans = bad[word]; spans != 0; spans &= spans - 1) {
      const int tile = (32 * word + __ffs(spans) - 1) * per, end = min((tile + per) * kKeys, last + 1);
      for (int d = from; d < width; d += d % 2 ? 7 : 1) {
        float sum = 0.f;
        for (int j = tile * kKeys; j < end; j += kAtOnce) {
          float x[kAtOnce];
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) x[u] = j + u < end ? __ldg(v + (j + u) * v_token + d) : 0.f;
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) sum += fabsf(x[u]) < INFINITY ? 0.f : x[u];
        }
        if (sum != 0.f) out[d] += sum;
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(F32Shape<D>::kThreads, D > 64 ? 1 : D > 32 ? 2 : 3) cow_prompt_f32_kernel(const __grid_constant__ PromptLaunch P) {
  using S = F32Shape<D>;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint16_t* s_q = reinterpret_cast<uint16_t*>(smem_raw);  // [3][kRows][kStride] bf16 parts
  uint16_t* s_k = s_q + 3 * S::kRows * S::kStride;         // [3][kKeys][kStride]
  uint16_t* s_v = s_k + 3 * kKeys * S::kStride;             // [3][kKeys][kStride]
  __shared__ Tile s_tile;
  __shared__ unsigned s_bad[kBadWords];  // spans of key tiles with values that are not finite
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int group = P.group, tile_tokens = S::kRows / group, kv_head = blockIdx.x % P.kv_heads, W = P.width;
  const float* Q = static_cast<const float*>(P.q);
  const float* K = static_cast<const float*>(P.k) + kv_head * P.k_head;
  const float* V = static_cast<const float*>(P.v) + kv_head * P.v_head;
  if (warp == 0) {
    TileFinder finder;
    finder.begin(P, tile_tokens);
    const Tile t = finder.find(P, tile_tokens, blockIdx.x / P.kv_heads);
    if (lane == 0) s_tile = t;
    if (lane < kBadWords) s_bad[lane] = 0;
  }
  __syncthreads();
  const Tile t = s_tile;
  if (t.count == 0) return;
  const int here = min(tile_tokens, t.count - t.first);  // tokens of this tile
  const int last = t.first + here;                       // keys 0 .. last - 1
  const int span = (last - 1) / (kKeys * 32 * kBadWords) + 1;  // key tiles to a bit of s_bad

  float4 k[S::kVecs], v[S::kVecs];
  auto load = [&](int j0) {
#pragma unroll
    for (int i = 0; i < S::kVecs; ++i) {
      const int n = tid + i * S::kThreads, r = n / (D / 4), d = 4 * (n % (D / 4));
      k[i] = v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j0 + r < last && d < W) {
        const int64_t token = t.begin + j0 + r;
        k[i] = __ldg(reinterpret_cast<const float4*>(K + token * P.k_token + d));
        v[i] = __ldg(reinterpret_cast<const float4*>(V + token * P.v_token + d));
      }
    }
  };
  load(0);
  // queries: a warp's own 16 rows, kLanes lanes to a row, all loads under way before the first is used
  {
    constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes, kTurns = 16 / kAtOnce;
    const int sub = lane / kLanes, d = 4 * (lane % kLanes);
    float4 x[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int r = 16 * warp + i * kAtOnce + sub, token = r / group;
      x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (token < here && d < W)
        x[i] = __ldg(reinterpret_cast<const float4*>(Q + (t.begin + t.first + token) * P.q_token +
                                                     (static_cast<int64_t>(kv_head) * group + r % group) * P.q_head + d));
    }
    // The scale is in the queries: scores less their maximum are then exact, where a product with the scale, rounded in the
    // maximum alone, would put the weights of scores above 2^31 beyond the type.
    const uint64_t scale = pair(P.scale_log2, P.scale_log2);
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const uint3 a = split3(mul2(pair(x[i].x, x[i].y), scale)), b = split3(mul2(pair(x[i].z, x[i].w), scale));
      uint16_t* to = s_q + (16 * warp + i * kAtOnce + sub) * S::kStride + d;
      *reinterpret_cast<uint2*>(to) = make_uint2(a.x, b.x);
      *reinterpret_cast<uint2*>(to + S::kRows * S::kStride) = make_uint2(a.y, b.y);
      *reinterpret_cast<uint2*>(to + 2 * S::kRows * S::kStride) = make_uint2(a.z, b.z);
    }
  }
  __syncwarp();
  const int row0 = 16 * warp + g;  // this lane's rows: row0 and row0 + 8
  const int query0 = t.first + row0 / group, query1 = t.first + (row0 + 8) / group;  // their places in the sequence

  float o[D / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  for (int j0 = 0; j0 < last; j0 += kKeys) {
    float mk = 0.f, mv = 0.f;  // whether all of them are finite
#pragma unroll
    for (int i = 0; i < S::kVecs; ++i) {
      mk = max3_nan(max3_nan(mk, fabsf(k[i].x), fabsf(k[i].y)), fabsf(k[i].z), fabsf(k[i].w));
      mv = max3_nan(max3_nan(mv, fabsf(v[i].x), fabsf(v[i].y)), fabsf(v[i].z), fabsf(v[i].w));
    }
    const bool odd_k = !(mk < INFINITY);
    if (!(mv < INFINITY)) {  // seldom: values that are not finite are left out
      auto finite = [](float x) { return fabsf(x) < INFINITY ? x : 0.f; };
#pragma unroll
      for (int i = 0; i < S::kVecs; ++i) v[i] = make_float4(finite(v[i].x), finite(v[i].y), finite(v[i].z), finite(v[i].w));
      const int at = j0 / kKeys / span;
      atomicOr(&s_bad[at / 32], 1u << (at % 32));
    }
    __syncthreads();  // the last tile is used up
#pragma unroll
    for (int i = 0; i < S::kVecs; ++i) {
      const int n = tid + i * S::kThreads, at = n / (D / 4) * S::kStride + 4 * (n % (D / 4));
      auto put = [&](uint16_t* to, float4 f) {
        const uint3 a = split3(pair(f.x, f.y)), b = split3(pair(f.z, f.w));
        *reinterpret_cast<uint2*>(to) = make_uint2(a.x, b.x);
        *reinterpret_cast<uint2*>(to + kKeys * S::kStride) = make_uint2(a.y, b.y);
        *reinterpret_cast<uint2*>(to + 2 * kKeys * S::kStride) = make_uint2(a.z, b.z);
      };
      put(s_k + at, k[i]);
      put(s_v + at, v[i]);
    }
    if (odd_k) {  // what is not finite of a key is its third part, which meets the queries' first alone: parts of unlike signs would make it NaN
#pragma unroll
      for (int i = 0; i < S::kVecs; ++i) {
        const int n = tid + i * S::kThreads, at = n / (D / 4) * S::kStride + 4 * (n % (D / 4));
        const float e[4] = {k[i].x, k[i].y, k[i].z, k[i].w};
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (!(fabsf(e[u]) < INFINITY)) {
            s_k[at + u] = s_k[kKeys * S::kStride + at + u] = 0;
            s_k[2 * kKeys * S::kStride + at + u] = static_cast<uint16_t>(pack_bf162(e[u], 0.f));
          }
      }
    }
    __syncthreads();
    if (j0 + kKeys < last) load(j0 + kKeys);

    // Scores: 16 rows x 64 keys.  The matrix unit cuts sums off where f32 rounds them, so the small products are added up first
    // and those of the first parts, which every later cut would be measured by, last.
    float s[8][4] = {};
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
      for (int d = 0; d < D; d += 16) {
        if (d >= W) break;
        unsigned q[3][4];
        const uint16_t* at = s_q + (16 * warp + (lane & 15)) * S::kStride + d + (lane >> 4) * 8;
#pragma unroll
        for (int y = 0; y < (pass ? 1 : 3); ++y) load_matrices(q[y], at + y * S::kRows * S::kStride);
#pragma unroll
        for (int n = 0; n < 4; n += 2) {  // 32 keys: four sums take turns, as each product waits for the last of its sum
          unsigned b[3][8];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint16_t* to = s_k + (16 * (n + x) + (lane & 7) + (lane >> 4) * 8) * S::kStride + d + (lane >> 3 & 1) * 8;
#pragma unroll
            for (int y = 0; y < (pass ? 1 : 3); ++y) load_matrices(b[y] + 4 * x, to + y * kKeys * S::kStride);
          }
#pragma unroll
          for (int y = pass ? 0 : 2; y >= (pass ? 0 : 1); --y)  // parts y apart in all
#pragma unroll
            for (int z = 0; z <= y; ++z)
#pragma unroll
              for (int x = 0; x < 4; ++x) mma_bf16(s[2 * n + x], q[y - z], b[z][2 * x], b[z][2 * x + 1]);
        }
      }
    }
    // softmax: columns 8 n + 2 c and the next of rows row0, row0 + 8
    if (j0 + kKeys - 1 > t.first) {
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int key = j0 + 8 * n + 2 * c;
        if (key > query0) s[n][0] = -INFINITY;
        if (key + 1 > query0) s[n][1] = -INFINITY;
        if (key > query1) s[n][2] = -INFINITY;
        if (key + 1 > query1) s[n][3] = -INFINITY;
      }
    }
    float big0 = -INFINITY, big1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      big0 = fmaxf(big0, fmaxf(s[n][0], s[n][1]));
      big1 = fmaxf(big1, fmaxf(s[n][2], s[n][3]));
    }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      big0 = fmaxf(big0, __shfl_xor_sync(kFull, big0, x));
      big1 = fmaxf(big1, __shfl_xor_sync(kFull, big1, x));
    }
    const float n0 = fmaxf(m0, big0 + kHeadroom), n1 = fmaxf(m1, big1 + kHeadroom);
    const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;  // all -inf so far: weights 0
    const float a0 = exp2_fast(m0 - b0), a1 = exp2_fast(m1 - b1);
    m0 = n0;
    m1 = n1;
    l0 *= a0;
    l1 *= a1;
    const uint64_t b00 = pair(-b0, -b0), b11 = pair(-b1, -b1);
    uint64_t e0[8], e1[8], sum0 = pair(0.f, 0.f), sum1 = sum0;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const float2 y0 = both(add2(pair(s[n][0], s[n][1]), b00)), y1 = both(add2(pair(s[n][2], s[n][3]), b11));
      e0[n] = pair(exp2_fast(y0.x), exp2_fast(y0.y));
      e1[n] = pair(exp2_fast(y1.x), exp2_fast(y1.y));
      sum0 = add2(sum0, e0[n]);
      sum1 = add2(sum1, e1[n]);
    }
    l0 += both(sum0).x + both(sum0).y;
    l1 += both(sum1).x + both(sum1).y;
    unsigned p[3][4][4];  // parts, by 16 keys
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const uint3 u = split3(e0[n]), w = split3(e1[n]);
      p[0][n / 2][2 * (n % 2)] = u.x;
      p[0][n / 2][2 * (n % 2) + 1] = w.x;
      p[1][n / 2][2 * (n % 2)] = u.y;
      p[1][n / 2][2 * (n % 2) + 1] = w.y;
      p[2][n / 2][2 * (n % 2)] = u.z;
      p[2][n / 2][2 * (n % 2) + 1] = w.z;
    }
#pragma unroll
    for (int d = 0; d < D; d += 32) {
      if (d >= W) break;
      // The tile's sum apart, then added in f32: the matrix unit's own adds do not round to nearest, and over
      // a long prompt that would show.
      float y4[4][4] = {};
#pragma unroll
      for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          unsigned b[3][8];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint16_t* at = s_v + (16 * n + (lane & 15)) * S::kStride + d + 16 * x + (lane >> 4) * 8;
#pragma unroll
            for (int y = 0; y < (pass ? 1 : 3); ++y) load_matrices_turned(b[y] + 4 * x, at + y * kKeys * S::kStride);
          }
#pragma unroll
          for (int y = pass ? 0 : 2; y >= (pass ? 0 : 1); --y)
#pragma unroll
            for (int z = 0; z <= y; ++z)
#pragma unroll
              for (int x = 0; x < 4; ++x) mma_bf16(y4[x], p[y - z][n], b[z][2 * x], b[z][2 * x + 1]);
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float* to = o[d / 8 + x];
        to[0] = fmaf(to[0], a0, y4[x][0]);
        to[1] = fmaf(to[1], a0, y4[x][1]);
        to[2] = fmaf(to[2], a1, y4[x][2]);
        to[3] = fmaf(to[3], a1, y4[x][3]);
      }
    }
  }
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    l0 += __shfl_xor_sync(kFull, l0, x);
    l1 += __shfl_xor_sync(kFull, l1, x);
  }
  unsigned bad = 0;
#pragma unroll
  for (int i = 0; i < kBadWords; ++i) bad |= s_bad[i];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = row0 + 8 * half, token = r / group, query = half ? query1 : query0;
    if (token >= here || r >= tile_tokens * group) continue;
    const float inv = 1.f / (half ? l1 : l0);
    float* out = static_cast<float*>(P.out) +
                 (static_cast<int64_t>(t.begin + query) * P.heads + static_cast<int64_t>(kv_head) * group + r % group) * W;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const int d = 8 * i + 2 * c;
      if (d >= W) continue;
      *reinterpret_cast<float2*>(out + d) = make_float2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
    }
    if (bad) add_nonfinite_f32(V + t.begin * P.v_token, P.v_token, s_bad, span, query, out, 2 * c, W);
  }
}

// --------------------------------------------------------------------------
// 16-bit types: tcgen05
// --------------------------------------------------------------------------
//
// A block, one to an SM, has two tiles A and B of 128 rows against key tiles of 128 tokens, twenty warps:
//   warps 0-7, 8-15  softmax of A and of B: two threads to a row, 64 keys each, so that the row's scores
//                    fit registers with four warps to a scheduler; the two meet once a key tile
//   warp 16          one thread loads by TMA: the query tiles once, K and V tiles round a ring
//   warp 17          one thread issues the products: S = Q K^T into tensor memory, and O += P V
//                    with P read from tensor memory, where it takes the place of S
//   warp 18          looks through the values of masked tiles (below)
//   warp 19          finds the next tiles
// While one tile's softmax runs, the tensor cores work on the other's O += P V and next S; S(j + 1) of a
// tile is issued after O += P V (j) of it, so its arrival also says that O may be touched.
// O lies in tensor memory for the whole pass.  It is rescaled only when a row's maximum has grown by more
// than 2^8 since the last time (P then still fits 16 bits and the sums are f32): by the softmax warps
// themselves, and seldom.  P is rounded to the input's type for the second product: the relative 2^-9 (2^-12
// for f16) of each weight averages out in the sum, and is of the size of the result's own rounding.
//
// Masked places: a weight of 0 times a value of infinity or NaN is NaN in a matrix product, so the values of
// tiles that any row sees only in part (of later tokens, and past the sequence's end of
// other sequences) are looked through first, non-finite ones are taken out, and rows that do see
// them have them added at the end.
//
// A block stays and takes tile after tile: loads and scores of the next begin under the end of the last.
// Measured (bf16): 2 x 8,192 tokens, 32/8 heads of 128: 1.00-1.03 ms, 1,070-1,100 TFLOP/s back to back under the power
// cap (a cuBLAS product sustains 1,384 there, 1,658 in a burst); 32 requests of 64 to 2,048, 16/4 heads of 64: 188-193 us,
// 530-550 TFLOP/s; 21 of 1 to 777, 14/2 heads of 96 (f16): 35-36 us.  Bound: the chain from a tile's scores through its softmax
// (1,750 cycles) and the two products (768 after the first half of P) back to its next scores, 2,900 cycles for the
// 2,048 of tensor work of both tiles; for narrow heads the 48 special-function and 370 other instructions of a warp for
// 32 rows of 64 keys; for short prompts what a tile costs beside its key tiles, 4,000 cycles (last products,
// 1,200; output, 2,000; next tile and its scores, 1,500, partly under the other tile's softmax).  Tried and not kept:
// a thread for each row with all 128 scores in registers (3,430 cycles a step), issue threads of A's and of B's own
// (they fall into step with each other: 4,200), three score tiles in turn for widths to 64 (the softmax is the
// bound: no change), the output given up as soon as it is in registers (the same: 1 % slower), masked tiles looked
// through only where some row does not see them, and from a step earlier (no change).
// Of eight pairs of weights, two come from the polynomial.  4,096 tokens of 16/4 heads of 32 / 64 / 96 / 128, us, with none,
// one, two and three: bf16 57 60 65 71, 53 56 60 64, 54 56 59 63, 56 58 62 67; f16 53 60 64 70, 52 56 61 65, 54 58 62 65,
// 56 61 65 67.
// Every wait is bounded; one that gives up sets a status bit and ends the block, all its rows NaN.

constexpr int kTcThreads = 640;
constexpr int kTcRows = 128;  // rows of a tile
constexpr int kTcKeys = 128;  // tokens of a key tile
constexpr int kTcLimit = 1 << 18;                        // tries of the waits at a block's end
constexpr unsigned long long kTcPatience = 2000000000ull;  // ns of the others
constexpr float kLazy = 8.f;  // log2 of the growth of a maximum that is let pass
constexpr float kFar = 16777216.f;  // half a last place of what is larger is 1 and more

template <int DT, int DP>  // DP: width rounded up to 32s
struct TcShape {
  static constexpr int kParts = (DP + 63) / 64;                        // 128-byte wide parts of a row
  static constexpr int kPartBytes = 128 * 128;                  // 128 rows of one part
  static constexpr int kTileBytes = kParts * kPartBytes;
  static constexpr int kSlots = DP > 64 ? 4 : 8;                // ring of K and V tiles
  // log2 of what weights lie below 1 (and up to kLazy above that): sums of bf16's largest values, which are f32's, do not
  // overflow before their division; f16's do not come near, and its weights have no range to spare.
  static constexpr float kUnder = DT == COW_BF16 ? 16.f : 0.f;
  static constexpr int kPoly = 2;                               // of 8 pairs of weights, those from the polynomial
  static constexpr int kStage = 16 * 1024;                      // 1 KB for each softmax warp: outputs on their way to rows
  static constexpr int kBytes = (2 + kSlots) * kTileBytes + kStage + 1024;
};

struct TcLaunch {
  PromptLaunch p;
  CUtensorMap q, k, v;
};

struct TcBarriers {
  uint64_t full[8], empty[8];         // the ring
  uint64_t tile_full[2], tile_empty[2];  // what to work on
  uint64_t q_full, q_empty;
  uint64_t s[2], p[2][2];             // scores are there; halves of the weights are
  uint64_t o_full[2], o_empty[2];     // the output is complete; is read
  uint64_t look[2], looked[2];        // a masked tile's values are there; are looked through (two such tiles at most)
  uint64_t drain;
};

// What a block works on: two tiles of rows of one key head.
struct TcTile {
  int begin, count, first, kv_head;  // count 0: no more
  int here_a, here_b;                // tokens
  int n_a, n_b;                      // key tiles
  int masked_from;                   // key tiles from here on are not seen whole by every row

  __device__ __forceinline__ int n() const { return max(n_a, n_b); }
};

// Two warps (64 threads) at named barrier `id`: whether `yes` holds in any of their threads; a plain meeting.
__device__ __forceinline__ bool any_of_two_warps(int id, bool yes) {
  unsigned any;
  asm volatile(
      "{ .reg .pred p, q; setp.ne.u32 p, %1, 0; barrier.cta.red.or.pred q, %2, 64, p; selp.u32 %0, 1, 0, q; }"
      : "=r"(any)
      : "r"(static_cast<unsigned>(yes)), "r"(id)
      : "memory");
  return any != 0;
}
__device__ __forceinline__ void two_warps_meet(int id) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory"); }

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ unsigned long long nanoseconds() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// A wait that was not over at once, out of line: the roles' code has to stay small for the instruction caches.
__device__ __noinline__ bool wait_long(uint64_t* bar, unsigned parity, volatile int* abort) {
  const unsigned long long since = nanoseconds();
  while (!mbar_wait(bar, parity, 64)) {
    if (*abort) return false;
    if (nanoseconds() - since > kTcPatience) {
      *abort = 1;
      return false;
    }
  }
  return true;
}

// One thread of a converged warp, known to the compiler to be one.
__device__ __forceinline__ bool elect_one() {
  unsigned one;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// D (tensor memory) (+)= A (shared memory) B (shared memory)
__device__ __forceinline__ void tc_mma_ss(unsigned d, uint64_t a, uint64_t b, unsigned idesc, bool add) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a),
      "l"(b), "r"(idesc), "r"(static_cast<unsigned>(add))
      : "memory");
}
// D (tensor memory) (+)= A (tensor memory) B (shared memory)
__device__ __forceinline__ void tc_mma_ts(unsigned d, unsigned a, uint64_t b, unsigned idesc, bool add) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a),
      "l"(b), "r"(idesc), "r"(static_cast<unsigned>(add))
      : "memory");
}

#define COW_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define COW_W8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
// 32 columns of this warp's 32 lanes of tensor memory, a lane's to its thread
__device__ __forceinline__ void tc_load32(unsigned at, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : COW_R8(r, 0), COW_R8(r, 8), COW_R8(r, 16), COW_R8(r, 24)
      : "r"(at));
}
// 16 columns, complete after tc_wait_loads16 of the same registers
__device__ __forceinline__ void tc_load16(unsigned at, unsigned* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : COW_R8(r, 0), COW_R8(r, 8)
               : "r"(at));
}
#define COW_RW8(a, i) "+r"(a[i]), "+r"(a[i + 1]), "+r"(a[i + 2]), "+r"(a[i + 3]), "+r"(a[i + 4]), "+r"(a[i + 5]), "+r"(a[i + 6]), "+r"(a[i + 7])
__device__ __forceinline__ void tc_wait_loads16(unsigned* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : COW_RW8(r, 0), COW_RW8(r, 8)::"memory");
}
#undef COW_RW8
__device__ __forceinline__ void tc_load8(unsigned at, unsigned* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : COW_R8(r, 0) : "r"(at));
}
__device__ __forceinline__ void tc_store8(unsigned at, const unsigned* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::COW_W8(r, 0), "r"(at) : "memory");
}
__device__ __forceinline__ void tc_store16(unsigned at, const unsigned* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::COW_W8(r, 0),
      COW_W8(r, 8), "r"(at)
      : "memory");
}
#undef COW_R8
#undef COW_W8
__device__ __forceinline__ void tc_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared memory operand, 128-byte swizzle, rows of 128 bytes, 8-row groups 1024 bytes apart.
// `lead`: for an operand whose rows are the contraction (values: a row is a token), bytes between 64-column parts.
__device__ __forceinline__ uint64_t operand_at(unsigned addr, unsigned lead) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
}

template <int DT>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  if constexpr (DT == COW_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
  }
}
// 2^y of both halves on the multiply-add pipe, for y <= about 100: with n the nearest integer, f = y - n in
// [-1/2, 1/2] and 2^f a polynomial with constant term 1, fitted here by reweighted least squares to
// the relative error (degree 3: 1.0e-4, degree 4: 2.8e-6, below the rounding of a weight to bf16, f16).
// Exactly 0 at and below y = -127, where a masked place's -inf ends up.
template <int DT>
__device__ __forceinline__ float2 exp2_poly(uint64_t y2) {
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, held in the low bits
  float2 y = both(y2);
  y2 = pair(fmaxf(y.x, -127.f), fmaxf(y.y, -127.f));
  const uint64_t t = add2(y2, pair(kMagic, kMagic));
  const uint64_t f = fma2(add2(t, pair(-kMagic, -kMagic)), pair(-1.f, -1.f), y2);
  uint64_t p;
  if constexpr (DT == COW_BF16) {
    p = fma2(f, pair(0.05500892922282219f, 0.05500892922282219f), pair(0.2422109693288803f, 0.2422109693288803f));
    p = fma2(p, f, pair(0.6932829022407532f, 0.6932829022407532f));
  } else {
    p = fma2(f, pair(0.009582852944731712f, 0.009582852944731712f), pair(0.055906426161527634f, 0.055906426161527634f));
    p = fma2(p, f, pair(0.24024099111557007f, 0.24024099111557007f));
    p = fma2(p, f, pair(0.6931241750717163f, 0.6931241750717163f));
  }
  p = fma2(p, f, pair(1.f, 1.f));
  const float2 r = both(p), n = both(t);
  return make_float2(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(n.x) << 23)),
                     __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(n.y) << 23)));
}

// 0 * w + sum of two 16-bit values
template <int DT>
__device__ __forceinline__ unsigned zero_times(unsigned w, unsigned sum) {
  unsigned r;
  if constexpr (DT == COW_BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(sum));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(sum));
  return r;
}

// Adds to a row's output the values of tokens first..last that are not finite: those of every 16 columns of
// two, from column `from` on.
template <int DT>
__device__ __noinline__ void add_nonfinite(const PromptLaunch& P, int first, int last, int kv_head, uint16_t* out, int from) {
  auto value = [](uint16_t u) {
    return DT == COW_BF16 ? __uint_as_float(static_cast<unsigned>(u) << 16) : __half2float(*reinterpret_cast<const __half*>(&u));
  };
  for (int d = from; d < P.width; d += d % 16 == 15 ? 17 : 1) {
    float sum = value(out[d]);
    for (int j = first; j <= last; ++j) {
      const float f = value(static_cast<const uint16_t*>(P.v)[j * P.v_token + kv_head * P.v_head + d]);
      if (!(fabsf(f) < INFINITY)) sum += f;
    }
    out[d] = static_cast<uint16_t>(pack2<DT>(sum, 0.f));
  }
}

// What a block works on at place i of its own order: back and forth over the blocks, so that each gets large and small tiles.
__device__ __forceinline__ int place_of(int i) { return i * gridDim.x + (i & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x); }

// A wait gave up: every row of the block's tiles becomes NaN, those it had not come to among them.  By all warps.
__device__ __noinline__ void give_up_rows(const PromptLaunch& P, int tile_tokens) {
  const int lane = threadIdx.x & 31;
  TileFinder finder;
  finder.begin(P, tile_tokens);
  for (int i = threadIdx.x >> 5;; i += kTcThreads / 32) {
    const int w = place_of(i);
    const Tile t = finder.find(P, tile_tokens, w / P.kv_heads);
    if (t.count == 0) return;
    const int row = P.group * P.width, here = min(tile_tokens, t.count - t.first);
    for (int token = 0; token < here; ++token) {
      uint16_t* out = static_cast<uint16_t*>(P.out) +
                      (static_cast<int64_t>(t.begin + t.first + token) * P.heads + static_cast<int64_t>(w % P.kv_heads) * P.group) * P.width;
      for (int d = lane; d < row; d += 32) out[d] = 0x7fff;  // NaN in either type
    }
  }
}

template <int DT, int DP>
__global__ void __launch_bounds__(kTcThreads, 1) cow_prompt_tc_kernel(const __grid_constant__ TcLaunch L) {
  using S = TcShape<DT, DP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ TcBarriers bars;
  __shared__ TcTile s_tiles[2];
  __shared__ int s_bad[2];
  __shared__ unsigned s_tmem;
  __shared__ int s_abort;
  __shared__ float s_most[2][2][kTcRows];
  const PromptLaunch& P = L.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = P.group, tile_tokens = kTcRows / group;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem;  // tiles A and B
  uint8_t* s_ring = smem + 2 * S::kTileBytes;
  uint8_t* s_stage = s_ring + S::kSlots * S::kTileBytes;

  if (warp == 16) {
    if (elect_one()) {
      prefetch_map(&L.q);
      prefetch_map(&L.k);
      prefetch_map(&L.v);
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (warp == 17 && lane == 0) {
    s_abort = 0;
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.tile_full[i], 1);
      mbar_init(&bars.tile_empty[i], 19);  // loads, products, looking through, 16 softmax warps
      mbar_init(&bars.s[i], 1);
      mbar_init(&bars.p[i][0], 8);
      mbar_init(&bars.p[i][1], 8);
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.o_empty[i], 8);
      mbar_init(&bars.look[i], 1);
      mbar_init(&bars.looked[i], 1);
    }
    mbar_init(&bars.drain, 1);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = s_tmem;
  auto wait = [&](uint64_t* bar, unsigned parity) { return mbar_wait(bar, parity, 1) || wait_long(bar, parity, &s_abort); };
  // the i-th of this block's tiles; false: none left, or a wait gave up
  auto next_tile = [&](int i, TcTile& t) {
    if (!wait(&bars.tile_full[i & 1], (i >> 1) & 1)) return false;
    t = s_tiles[i & 1];
    return t.count > 0;
  };

  if (warp == 19) {
    // ---- what to work on: tiles in the order of their work
    TileFinder finder;
    finder.begin(P, 2 * tile_tokens);
    for (int i = 0;; ++i) {
      const int w = place_of(i);
      const Tile f = finder.find(P, 2 * tile_tokens, w / P.kv_heads);
      if (i >= 2 && !__all_sync(kFull, wait(&bars.tile_empty[i & 1], ((i >> 1) - 1) & 1))) break;
      if (lane == 0) {
        TcTile t;
        t.begin = f.begin;
        t.count = f.count;
        t.first = f.first;
        t.kv_head = w % P.kv_heads;
        t.here_a = min(tile_tokens, f.count - f.first);
        t.here_b = max(min(tile_tokens, f.count - f.first - tile_tokens), 0);
        t.n_a = (f.first + t.here_a + kTcKeys - 1) / kTcKeys;
        t.n_b = t.here_b > 0 ? (f.first + tile_tokens + t.here_b + kTcKeys - 1) / kTcKeys : 0;
        t.masked_from = f.first / kTcKeys;
        s_tiles[i & 1] = t;
        s_bad[i & 1] = 0;
        mbar_arrive(&bars.tile_full[i & 1]);
      }
      if (f.count == 0) break;
    }
  } else if (warp == 16 && elect_one()) {
    // ---- loads
    TcTile t;
    int item = 0, tiles = 0;  // tiles of K and V, and of queries, so far
    bool ok = true;
    for (; ok && next_tile(tiles, t); ++tiles) {
      auto load = [&](int i) {  // K(0), V(0), K(1), ...
        const int slot = item % S::kSlots;
        if (item >= S::kSlots && !wait(&bars.empty[slot], (item / S::kSlots - 1) & 1)) return false;
        mbar_arrive_expect_tx(&bars.full[slot], S::kTileBytes);
        for (int part = 0; part < S::kParts; ++part)
          tma_load(s_ring + slot * S::kTileBytes + part * S::kPartBytes, i & 1 ? &L.v : &L.k, 64 * part, t.kv_head,
                   t.begin + (i >> 1) * kTcKeys, &bars.full[slot]);
        ++item;
        return true;
      };
      ok = load(0) && (tiles == 0 || wait(&bars.q_empty, (tiles - 1) & 1));
      if (!ok) break;
      const int both_tiles = t.here_b > 0 ? 2 : 1;
      mbar_arrive_expect_tx(&bars.q_full, both_tiles * S::kParts * 128 * group * tile_tokens);
      for (int x = 0; x < both_tiles; ++x)
        for (int part = 0; part < S::kParts; ++part)
          tma_load(s_q + x * S::kTileBytes + part * S::kPartBytes, &L.q, 64 * part, t.kv_head * group,
                   t.begin + t.first + x * tile_tokens, &bars.q_full);
      const int n = t.n();
      for (int i = 1; ok && i < 2 * n; ++i) ok = load(i);
      mbar_arrive(&bars.tile_empty[tiles & 1]);
    }
    // nothing may still be on its way into shared memory when the block ends
    if (tiles > 0) mbar_wait(&bars.q_full, (tiles - 1) & 1, kTcLimit);
    if (!ok) mbar_wait(&bars.q_full, tiles & 1, 4096);  // the tile that was broken off, if it got that far
    for (int i = max(item - S::kSlots, 0); i < item; ++i) mbar_wait(&bars.full[i % S::kSlots], (i / S::kSlots) & 1, kTcLimit);
  } else if (warp == 17 && elect_one()) {
    // ---- products
    constexpr int kSteps = DP / 16;
    constexpr unsigned kType = DT == COW_BF16 ? 1u : 0u;
    const unsigned base = (1u << 4) | (kType << 7) | (kType << 10) | ((128u >> 4) << 24);
    // S: 128 x 128, both operands contiguous along the width; a negative scale negates Q
    const unsigned idesc_s = base | ((128u >> 3) << 17) | (P.scale_log2 < 0.f ? 1u << 13 : 0u);
    // O: 128 x width, values contiguous along the output's columns
    const unsigned idesc_o = base | (1u << 16) | (static_cast<unsigned>(2 * kSteps) << 17);
    const uint64_t desc_q = operand_at(smem_addr(s_q), 16), desc_ring = operand_at(smem_addr(s_ring), 16);
    const uint64_t desc_v = operand_at(smem_addr(s_ring), S::kPartBytes);
    TcTile t;
    int item = 0;                                  // the tile's K(0) in the count of all K and V tiles
    unsigned steps[2] = {0, 0}, done[2] = {0, 0};  // key tiles, and tiles of rows, of A and of B so far
    unsigned looks[2] = {0, 0};
    bool ok = true;
    for (int tiles = 0; ok && next_tile(tiles, t); ++tiles) {
      const int n = t.n();
      auto score = [&](int x, int j) {
        const uint64_t q = desc_q + x * (S::kTileBytes >> 4), k = desc_ring + ((item + 2 * j) % S::kSlots) * (S::kTileBytes >> 4);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int off = ((i / 4) * S::kPartBytes + (i % 4) * 32) >> 4;
          tc_mma_ss(tmem + 128 * x, q + off, k + off, idesc_s, i > 0);
        }
        tc_commit(&bars.s[x]);
      };
      auto output = [&](int x, int j, int h) {  // of each half of the tile's tokens, its half h
        const uint64_t v = desc_v + ((item + 2 * j + 1) % S::kSlots) * (S::kTileBytes >> 4);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tc_mma_ts(tmem + 256 + 128 * x, tmem + 128 * x + 64 * (i / 2) + 16 * h + 8 * (i % 2),
                    v + (2048 >> 4) * (4 * (i / 2) + 2 * h + i % 2), idesc_o, j > 0 || h > 0 || i > 0);
      };
      auto full = [&](int i) { return wait(&bars.full[(item + i) % S::kSlots], ((item + i) / S::kSlots) & 1); };
      // V(j) is there; a masked tile's values are looked through
      auto values = [&](int j) {
        if (j >= n) return true;
        if (!full(2 * j + 1)) return false;
        if (j >= t.masked_from) mbar_arrive(&bars.look[j - t.masked_from]);
        return true;
      };
      ok = full(0) && wait(&bars.q_full, tiles & 1);
      if (ok) {
        tc_fence_after();
        score(0, 0);
        if (t.n_b > 0) score(1, 0);
        tc_commit(&bars.empty[item % S::kSlots]);
        if (n == 1) tc_commit(&bars.q_empty);
        ok = values(0) && (n == 1 || full(2));
      }
      for (int j = 0; ok && j < n; ++j) {
        if (j >= t.masked_from) {
          const int k = j - t.masked_from;
          ok = wait(&bars.looked[k], looks[k] & 1);
          ++looks[k];
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int nx = x ? t.n_b : t.n_a;
          if (ok && j < nx) {
            const unsigned phase = steps[x] & 1;
            ++steps[x];
            // the previous tile's output must have been read before the first product of this one's
            ok = (j > 0 || done[x] == 0 || wait(&bars.o_empty[x], (done[x] - 1) & 1)) && wait(&bars.p[x][0], phase);
            if (ok) {
              tc_fence_after();
              output(x, j, 0);
              ok = wait(&bars.p[x][1], phase);
            }
            if (ok) {
              tc_fence_after();
              output(x, j, 1);
              if (j + 1 < nx) {
                score(x, j + 1);
              } else {
                tc_commit(&bars.o_full[x]);
                ++done[x];
              }
            }
          }
          if (x == 0) ok = ok && values(j + 1);  // while B's softmax is at work
        }
        ok = ok && (j + 2 >= n || full(2 * j + 4));  // K(j + 2), while A's is
        if (ok) {
          tc_commit(&bars.empty[(item + 2 * j + 1) % S::kSlots]);
          if (j + 1 < n) tc_commit(&bars.empty[(item + 2 * j + 2) % S::kSlots]);
          if (j + 2 == n) tc_commit(&bars.q_empty);  // the last scores are issued
        }
      }
      item += 2 * n;
      if (ok) mbar_arrive(&bars.tile_empty[tiles & 1]);
    }
    // products in flight end before tensor memory is given back
    tc_commit(&bars.drain);
    mbar_wait(&bars.drain, 0, kTcLimit);
  } else if (warp == 18) {
    // ---- values of masked tiles
    TcTile t;
    int item = 0;
    unsigned looks[2] = {0, 0};
    bool ok = true;
    for (int tiles = 0; ok && __all_sync(kFull, next_tile(tiles, t)); ++tiles) {
      const int n = t.n();
      for (int j = t.masked_from; ok && j < n; ++j) {
        const int k = j - t.masked_from, i = item + 2 * j + 1;
        ok = __all_sync(kFull, wait(&bars.look[k], looks[k] & 1) && wait(&bars.full[i % S::kSlots], (i / S::kSlots) & 1));
        if (!ok) break;
        ++looks[k];
        uint4* words = reinterpret_cast<uint4*>(s_ring + (i % S::kSlots) * S::kTileBytes);
        constexpr int kEach = S::kTileBytes / 16 / 32;
        unsigned sum[4] = {};  // of 0 times each value, by halves: NaN once one is not finite; four, as each waits for its last
#pragma unroll 8
        for (int u = 0; u < kEach; ++u) {
          const uint4 w = words[u * 32 + lane];
          sum[0] = zero_times<DT>(w.x, sum[0]);
          sum[1] = zero_times<DT>(w.y, sum[1]);
          sum[2] = zero_times<DT>(w.z, sum[2]);
          sum[3] = zero_times<DT>(w.w, sum[3]);
        }
        if (((sum[0] | sum[1] | sum[2] | sum[3]) & 0x7fff7fffu) != 0) {
          constexpr unsigned kExp = DT == COW_BF16 ? 0x7f80u : 0x7c00u;
          s_bad[tiles & 1] = 1;
          for (int u = 0; u < kEach; ++u) {
            unsigned* w = reinterpret_cast<unsigned*>(words + u * 32 + lane);
            for (int y = 0; y < 4; ++y) {
              if ((w[y] & kExp) == kExp) w[y] &= 0xffff0000u;
              if (((w[y] >> 16) & kExp) == kExp) w[y] &= 0xffffu;
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.looked[k]);
      }
      item += 2 * n;
      if (ok && lane == 0) mbar_arrive(&bars.tile_empty[tiles & 1]);
    }
  } else if (warp < 16) {
    // ---- softmax
    const int x = warp >> 3, half = (warp >> 2) & 1;  // this thread's half of the keys
    const int row = tid & 127, row_token = row / group, row_head = row - row_token * group;
    uint4* stage = reinterpret_cast<uint4*>(s_stage + warp * 1024);  // 32 rows of two 16-byte words
    const unsigned lanes = tmem + (static_cast<unsigned>(warp & 3) << 21);  // this warp's 32 lanes
    const unsigned at_s = lanes + 128 * x + 64 * half, at_o = lanes + 256 + 128 * x;
    const int meet = 1 + 4 * x + (warp & 3);  // the barrier of the two warps that share 32 rows
    const float c = fabsf(P.scale_log2);
    unsigned steps = 0, done = 0;
    bool ok = true;
    for (int tiles = 0;; ++tiles) {
      // A wait that gave up is only remembered: both warps of a pair go on to their common end of the tile.
      if (any_of_two_warps(meet, !ok || !wait(&bars.tile_full[tiles & 1], (tiles >> 1) & 1))) break;
      const TcTile& t = s_tiles[tiles & 1];
      if (t.count == 0) break;
      const int nx = x ? t.n_b : t.n_a;
      const int first = t.first + x * tile_tokens, query = first + row_token;  // its place in the sequence
      bool far = false;              // for any row of the warp: see kFar
      float m = -INFINITY, l = 0.f;  // m: the score that P is relative to, the same in both halves
      for (int j = 0; j < nx; ++j, ++steps) {
        ok = __all_sync(kFull, wait(&bars.s[x], steps & 1)) && ok;
        tc_fence_after();
        unsigned s[64];
        tc_load32(at_s, s);
        tc_load32(at_s + 32, s + 32);
        tc_wait_loads();
        if (j * kTcKeys + kTcKeys - 1 > first) {
          const int seen = query - j * kTcKeys - 64 * half;
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i > seen) s[i] = 0xff800000u;
        }
        float big[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) big[i] = __uint_as_float(s[i]);
#pragma unroll
        for (int i = 4; i < 64; i += 2) {
          float& b = big[(i / 2) & 3];
          b = max3_nan(b, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        }
        float now = max3_nan(max3_nan(big[0], big[1], big[2]), big[3], big[3]);
        if (any_of_two_warps(meet, !((now - m) * c <= kLazy))) {  // NaN too
          s_most[x][half][row] = now;
          two_warps_meet(meet);
          now = max3_nan(now, s_most[x][half ^ 1][row], m);
          const bool grown = !((now - m) * c <= kLazy);
          float next = grown ? now : m;
          if (next == INFINITY) next = __int_as_float(0x7fc00000);  // inf - inf: the row is NaN, as any that sees one
          const float a = next == -INFINITY ? 1.f : exp2_fast((m - next) * c);
          m = next;
          l *= a;
          if (j > 0) {
#pragma unroll 1
            for (int i = 8 * half; i < DP; i += 16) {  // few registers: the scores wait in theirs
              unsigned o[8];
              tc_load8(at_o + i, o);
              tc_wait_loads();
#pragma unroll
              for (int u = 0; u < 8; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * a);
              tc_store8(at_o + i, o);
            }
            tc_wait_stores();
          }
          far = __any_sync(kFull, row_token < tile_tokens && fabsf(m * c) > kFar && m != -INFINITY);
          two_warps_meet(meet);  // both have rescaled, and read the other's maximum
        }
        float base = m == -INFINITY ? 0.f : fmaf(m, c, S::kUnder);  // all -inf so far: weights 0
        // The maximum times the scale is rounded, a score's product below is not: where that alone would drive weights out of
        // range, the scores of the row are taken less their maximum first.  (From tensor memory, in few instructions.)
        if (far) {
          const int seen = query - j * kTcKeys - 64 * half;
          const bool mine = fabsf(base) > kFar;
          const float away = mine ? m : 0.f;
#pragma unroll 1
          for (int i = 0; i < 64; i += 8) {
            unsigned r[8];
            tc_load8(at_s + i, r);
            tc_wait_loads();
#pragma unroll
            for (int u = 0; u < 8; ++u) r[u] = i + u > seen ? 0xff800000u : __float_as_uint(__uint_as_float(r[u]) - away);
            tc_store8(at_s + i, r);
          }
          tc_wait_stores();
          tc_load32(at_s, s);
          tc_load32(at_s + 32, s + 32);
          tc_wait_loads();
          if (mine) base = S::kUnder;
        }
        const uint64_t c2 = pair(c, c), base2 = pair(-base, -base);
        uint64_t sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          unsigned p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t y = fma2(pair(__uint_as_float(s[32 * h + 2 * i]), __uint_as_float(s[32 * h + 2 * i + 1])), c2, base2);
            float2 e;
            if (i % 8 < S::kPoly) {
              e = exp2_poly<DT>(y);
            } else {
              e = both(y);
              e.x = exp2_fast(e.x);
              e.y = exp2_fast(e.y);
            }
            sum[i & 1] = add2(sum[i & 1], pair(e.x, e.y));
            p[i] = pack2<DT>(e.x, e.y);
          }
          tc_store16(at_s + 16 * h, p);
          tc_wait_stores();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.p[x][h]);
        }
        const float2 sums = both(add2(sum[0], sum[1]));
        l += sums.x + sums.y;
      }
      if (nx > 0) {
        // The sums meet while the last products run; of a wait that gave up they make NaN.
        s_most[x][half][row] = ok ? l : __int_as_float(0x7fc00000);
        two_warps_meet(meet);
        l += s_most[x][half ^ 1][row];
        const bool store = row_token < (x ? t.here_b : t.here_a);
        const float whole = 1.f / l;
        uint16_t* out = static_cast<uint16_t*>(P.out) + (static_cast<int64_t>(t.begin + query) * P.heads +
                                                         static_cast<int64_t>(t.kv_head) * group + row_head) * P.width;
        // A thread's row would leave by 16 bytes to each of 32 places at a time: 16 columns of the warp's rows go
        // through shared memory instead and leave by two neighbouring words of 16 rows.  This lane's places:
        uint16_t* to[2];
#pragma unroll
        for (int y = 0; y < 2; ++y)
          to[y] = reinterpret_cast<uint16_t*>(__shfl_sync(kFull, store ? reinterpret_cast<unsigned long long>(out) : 0ull, 16 * y + lane / 2));
        const int at_w = 2 * lane, turn_w = lane >> 2 & 1, at_r = lane ^ (lane >> 3 & 1);
        ok = __all_sync(kFull, wait(&bars.o_full[x], done & 1)) && ok;
        ++done;
        tc_fence_after();
        const float inv = ok ? whole : __int_as_float(0x7fc00000);
        const uint64_t inv2 = pair(inv, inv);
        const bool bad = s_bad[tiles & 1];
#pragma unroll 1
        for (int n = 0; n < DP / 32; ++n) {
          unsigned r[16];
          tc_load16(at_o + 32 * n + 16 * half, r);
          tc_wait_loads16(r);
          unsigned w[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float2 f = both(mul2(pair(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1])), inv2));
            w[u] = pack2<DT>(f.x, f.y);
          }
          stage[at_w + turn_w] = make_uint4(w[0], w[1], w[2], w[3]);
          stage[at_w + (turn_w ^ 1)] = make_uint4(w[4], w[5], w[6], w[7]);
          __syncwarp();
          const int d = 32 * n + 16 * half + 8 * (lane & 1);
          if (d < P.width) {
#pragma unroll
            for (int y = 0; y < 2; ++y)
              if (to[y]) *reinterpret_cast<uint4*>(to[y] + d) = stage[32 * y + at_r];
          }
          __syncwarp();
        }
        tc_fence_before();
        if (lane == 0) mbar_arrive(&bars.o_empty[x]);
        if (bad && store)
          add_nonfinite<DT>(P, t.begin + t.masked_from * kTcKeys, t.begin + query, t.kv_head, out, 16 * half);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.tile_empty[tiles & 1]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  if (s_abort) {
    if (tid == 0 && P.status) atomicOr(P.status, COW_ST_WAIT_TIMEOUT);
    give_up_rows(P, 2 * tile_tokens);
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// [tokens][heads][width] of 16-bit elements in boxes of box_tokens x box_heads x 64
bool encode_rows(CUtensorMap* map, int dtype, const void* base, int64_t tokens, int64_t heads, int64_t width,
                 int64_t token_stride, int64_t head_stride, int box_tokens, int box_heads) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_stride) * 2, static_cast<cuuint64_t>(token_stride) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  const cuuint32_t ones[3] = {1, 1, 1};
  return fn(map, dtype == COW_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, int DP>
int launch_tc(const TcLaunch& L, unsigned blocks, cudaStream_t stream) {
  const int resident = resident_blocks(reinterpret_cast<const void*>(cow_prompt_tc_kernel<DT, DP>), kTcThreads, TcShape<DT, DP>::kBytes);
  if (!resident) return COW_ERR_CUDA;
  const unsigned grid = blocks < static_cast<unsigned>(resident) ? blocks : static_cast<unsigned>(resident);
  cow_prompt_tc_kernel<DT, DP><<<grid, kTcThreads, TcShape<DT, DP>::kBytes, stream>>>(L);
  return launch_status();
}

int prompt_tc(const PromptLaunch& P, cudaStream_t stream) {
  TcLaunch L;
  L.p = P;
  const int tile_tokens = kTcRows / P.group;
  if (!encode_rows(&L.q, P.dtype, P.q, P.tokens, P.heads, P.width, P.q_token, P.q_head, tile_tokens, P.group) ||
      !encode_rows(&L.k, P.dtype, P.k, P.tokens, P.kv_heads, P.width, P.k_token, P.k_head, kTcKeys, 1) ||
      !encode_rows(&L.v, P.dtype, P.v, P.tokens, P.kv_heads, P.width, P.v_token, P.v_head, kTcKeys, 1))
    return COW_ERR_INVALID;
  // every sequence adds at most one tile that is not full
  const int64_t tiles = P.tokens / (2 * tile_tokens) + (P.sequences < P.tokens ? P.sequences : P.tokens);
  const unsigned blocks = static_cast<unsigned>(tiles * P.kv_heads);
  const bool bf16 = P.dtype == COW_BF16;
  if (P.width <= 32) return bf16 ? launch_tc<COW_BF16, 32>(L, blocks, stream) : launch_tc<COW_F16, 32>(L, blocks, stream);
  if (P.width <= 64) return bf16 ? launch_tc<COW_BF16, 64>(L, blocks, stream) : launch_tc<COW_F16, 64>(L, blocks, stream);
  if (P.width <= 96) return bf16 ? launch_tc<COW_BF16, 96>(L, blocks, stream) : launch_tc<COW_F16, 96>(L, blocks, stream);
  return bf16 ? launch_tc<COW_BF16, 128>(L, blocks, stream) : launch_tc<COW_F16, 128>(L, blocks, stream);
}

template <int D>
int launch_f32(const PromptLaunch& P, cudaStream_t stream) {
  using S = F32Shape<D>;
  if (!resident_blocks(reinterpret_cast<const void*>(cow_prompt_f32_kernel<D>), S::kThreads, S::kBytes)) return COW_ERR_CUDA;
  // every sequence adds at most one tile that is not full
  const int64_t tiles = P.tokens / (S::kRows / P.group) + (P.sequences < P.tokens ? P.sequences : P.tokens);
  cow_prompt_f32_kernel<D><<<static_cast<unsigned>(tiles * P.kv_heads), S::kThreads, S::kBytes, stream>>>(P);
  return launch_status();
}

int prompt_f32(const PromptLaunch& P, cudaStream_t stream) {
  if (P.width <= 32) return launch_f32<32>(P, stream);
  return P.width <= 64 ? launch_f32<64>(P, stream) : launch_f32<128>(P, stream);
}

bool rows_ok(const void* p, int64_t s0, int64_t s1, int dtype) {
  const int64_t size = elem_size(dtype);
  return p && aligned16(p) && (s0 * size) % 16 == 0 && (s1 * size) % 16 == 0;
}

}  // namespace

extern "C" {

int cow_prompt_attention(const void* queries, int64_t query_token_stride, int64_t query_head_stride,
                         const void* keys, int64_t key_token_stride, int64_t key_head_stride, const void* values,
                         int64_t value_token_stride, int64_t value_head_stride, const int32_t* starts,
                         int64_t sequences, int64_t tokens, int32_t heads, int32_t kv_heads, int32_t width,
                         int32_t dtype, float scale, void* out, int32_t* status, void* stream) {
  if (!valid_dtype(dtype) || sequences < 0 || tokens < 0 || kv_heads < 1 || heads < 1 || heads % kv_heads || width < 1)
    return COW_ERR_INVALID;
  if (width % 8 || width > 128 || heads / kv_heads > kMaxGroup || tokens >= (int64_t{1} << 30) ||
      sequences >= (int64_t{1} << 30))
    return COW_ERR_UNSUPPORTED;
  if (sequences == 0 || tokens == 0) return COW_OK;
  if ((tokens / (kMaxGroup / (heads / kv_heads)) + (sequences < tokens ? sequences : tokens)) * kv_heads >= (int64_t{1} << 31))
    return COW_ERR_UNSUPPORTED;  // more blocks than one launch has
  if (!rows_ok(queries, query_token_stride, query_head_stride, dtype) ||
      !rows_ok(keys, key_token_stride, key_head_stride, dtype) ||
      !rows_ok(values, value_token_stride, value_head_stride, dtype) || !starts || !out || !aligned16(out))
    return COW_ERR_INVALID;
  // not 0, so that a masked score times it stays -inf
  const float scale_log2 = scale * 1.4426950408889634f;
  PromptLaunch P{queries, keys, values, out, starts, query_token_stride, query_head_stride, key_token_stride,
                 key_head_stride, value_token_stride, value_head_stride, status, static_cast<int32_t>(sequences),
                 static_cast<int32_t>(tokens), heads, kv_heads, heads / kv_heads, width, dtype,
                 fabsf(scale_log2) < kLeast ? kLeast : scale_log2};
  return dtype == COW_F32 ? prompt_f32(P, as_stream(stream)) : prompt_tc(P, as_stream(stream));
}

}  // extern "C"
