// cow_prompt.cu -- causal attention over packed prompts of different lengths, grouped heads.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale * q_i . k_j - m_i),   j <= i in i's own sequence
//
// A tile is kRows rows of one key head: neighbouring tokens times the key head's query heads, row =
// token * group + head, so that a group shares every key it reads and short prompts still fill
// their rows.  Keys pass in tiles of 64; maximum, sum and output of the running softmax stay in
// registers.  Tiles run in the order of their work, longest first, over all sequences
// together: the tile at place l of its sequence reads l + 1 tiles' keys, so the tiles of place l
// are one for each sequence that has more than l, and a block finds its own by a search
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
  int32_t sequences, tokens, heads, kv_heads, group, width, dtype;
  float scale_log2;  // scale * log2(e)
};

// Sequence b as [begin, begin + count), inside the packed tokens whatever `starts` holds.
__device__ __forceinline__ int2 sequence_of(const PromptLaunch& P, int b) {
  const int begin = min(max(P.starts[b], 0), P.tokens), end = min(max(P.starts[b + 1], begin), P.tokens);
  return make_int2(begin, end - begin);
}

struct Tile {
  int begin, count, first;  // its sequence, and its first token in it; count 0: none left
};

// The x-th tile of all in the order of work, found by one warp.
__device__ __forceinline__ Tile find_tile(const PromptLaunch& P, int tile_tokens, int x) {
  const int lane = threadIdx.x & 31;
  const int B = P.sequences;
  // tiles whose place is >= h
  auto above = [&](int h) {
    int n = 0;
    for (int b = lane; b < B; b += 32) n += max((sequence_of(P, b).y + tile_tokens - 1) / tile_tokens - h, 0);
    return __reduce_add_sync(kFull, n);
  };
  int most = 0;
  for (int b = lane; b < B; b += 32) most = max(most, (sequence_of(P, b).y + tile_tokens - 1) / tile_tokens);
  most = __reduce_max_sync(kFull, most);
  Tile t{0, 0, 0};
  if (x >= above(0)) return t;
  int lo = 0, hi = most;  // above(lo) > x >= above(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (above(mid) > x) lo = mid; else hi = mid;
  }
  int rank = x - above(hi);  // among the sequences with more than lo tiles
  for (int base = 0; base < B; base += 32) {
    int2 seq = make_int2(0, 0);
    if (base + lane < B) seq = sequence_of(P, base + lane);
    const unsigned has = __ballot_sync(kFull, (seq.y + tile_tokens - 1) / tile_tokens > lo);
    const int n = __popc(has);
    if (rank < n) {
      const int src = __fns(has, 0, rank + 1);
      t.begin = __shfl_sync(kFull, seq.x, src);
      t.count = __shfl_sync(kFull, seq.y, src);
      t.first = lo * tile_tokens;
      return t;
    }
    rank -= n;
  }
  return t;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// --------------------------------------------------------------------------
// f32 arithmetic
// --------------------------------------------------------------------------
//
// 64 rows against 64 keys at a time, 256 threads, each 4 x 4 scores and 4 rows x width / 16 of the output.

constexpr int kRows = 64;
constexpr int kKeys = 64;
constexpr int kThreads = 256;

template <int D>
__global__ void __launch_bounds__(kThreads) cow_prompt_f32_kernel(const __grid_constant__ PromptLaunch P) {
  constexpr int kStride = D + 4;
  constexpr int kCols = D / 16;
  extern __shared__ __align__(16) float smem_f[];
  float* s_q = smem_f;                     // [kRows][kStride]
  float* s_k = s_q + kRows * kStride;      // [kKeys][kStride]
  float* s_v = s_k + kKeys * kStride;      // [kKeys][kStride]
  float* s_p = s_v + kKeys * kStride;      // [kRows][kKeys + 4]
  __shared__ Tile s_tile;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int group = P.group, tile_tokens = kRows / group, kv_head = blockIdx.x % P.kv_heads, W = P.width;
  if (tid < 32) {
    const Tile t = find_tile(P, tile_tokens, blockIdx.x / P.kv_heads);
    if (tid == 0) s_tile = t;
  }
  __syncthreads();
  const Tile t = s_tile;
  if (t.count == 0) return;
  const int here = min(tile_tokens, t.count - t.first);  // tokens of this tile

  for (int i = tid; i < kRows * (D / 4); i += kThreads) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4)), token = r / group, h = r % group;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (token < here && d < W)
      x = ld4_rt(P.q, (t.begin + t.first + token) * P.q_token + (static_cast<int64_t>(kv_head) * group + h) * P.q_head + d, P.dtype);
    *reinterpret_cast<float4*>(s_q + r * kStride + d) = x;
  }
  float o[4][kCols], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < kCols; ++j) o[i][j] = 0.f;
  }
  const int last = t.first + here;  // keys 0 .. last - 1
  for (int j0 = 0; j0 < last; j0 += kKeys) {
    __syncthreads();
    for (int i = tid; i < kKeys * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = 4 * (i % (D / 4));
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      if (j0 + r < last && d < W) {
        const int64_t token = t.begin + j0 + r;
        a = ld4_rt(P.k, token * P.k_token + kv_head * P.k_head + d, P.dtype);
        b = ld4_rt(P.v, token * P.v_token + kv_head * P.v_head + d, P.dtype);
      }
      *reinterpret_cast<float4*>(s_k + r * kStride + d) = a;
      *reinterpret_cast<float4*>(s_v + r * kStride + d) = b;
    }
    __syncthreads();
    float s[4][4] = {};
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(s_q + (4 * ty + i) * kStride + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(s_k + (tx + 16 * j) * kStride + d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = fmaf(a[i].x, b[j].x, s[i][j]);
          s[i][j] = fmaf(a[i].y, b[j].y, s[i][j]);
          s[i][j] = fmaf(a[i].z, b[j].z, s[i][j]);
          s[i][j] = fmaf(a[i].w, b[j].w, s[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int query = t.first + (4 * ty + i) / group;  // its place in the sequence
      float big = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = j0 + tx + 16 * j <= query ? s[i][j] * P.scale_log2 : -INFINITY;
        big = fmaxf(big, s[i][j]);
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) big = fmaxf(big, __shfl_xor_sync(kFull, big, x));
      const float n = fmaxf(m[i], big), base = n == -INFINITY ? 0.f : n;
      const float a = exp2_fast(m[i] - base);
      m[i] = n;
      l[i] *= a;
#pragma unroll
      for (int j = 0; j < kCols; ++j) o[i][j] *= a;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2_fast(s[i][j] - base);
        l[i] += e;
        s_p[(4 * ty + i) * (kKeys + 4) + tx + 16 * j] = e;
      }
    }
    __syncwarp();  // a row's 16 threads are of one warp
    const int keys = min(kKeys, last - j0);
    for (int j = 0; j < keys; ++j) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = s_p[(4 * ty + i) * (kKeys + 4) + j];
        // a key after the query has no part in it, whatever its value (0 * inf is not 0)
        if (j0 + j > t.first + (4 * ty + i) / group) p[i] = 0.f;
      }
#pragma unroll
      for (int x = 0; x < kCols; ++x) {
        const float v = s_v[j * kStride + tx + 16 * x];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j0 + j <= t.first + (4 * ty + i) / group) o[i][x] = fmaf(p[i], v, o[i][x]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) l[i] += __shfl_xor_sync(kFull, l[i], x);
    const int r = 4 * ty + i, token = r / group, h = r % group;
    if (token >= here || r >= tile_tokens * group) continue;
    const float inv = 1.f / l[i];
    const int64_t row = (static_cast<int64_t>(t.begin + t.first + token) * P.heads + static_cast<int64_t>(kv_head) * group + h) * W;
#pragma unroll
    for (int x = 0; x < kCols; ++x) {
      const int d = tx + 16 * x;
      if (d >= W) continue;
      const float y = o[i][x] * inv;
      if (P.dtype == COW_F32) static_cast<float*>(P.out)[row + d] = y;
      else if (P.dtype == COW_BF16) static_cast<__nv_bfloat16*>(P.out)[row + d] = __float2bfloat16_rn(y);
      else static_cast<__half*>(P.out)[row + d] = __float2half_rn(y);
    }
  }
}

// --------------------------------------------------------------------------
// 16-bit types: tcgen05
// --------------------------------------------------------------------------
//
// A block has two tiles A and B of 128 rows against key tiles of 128 tokens, twelve warps:
//   warps 0-3, 4-7   softmax of A and of B: a thread owns a row, so maximum and sum need no exchange
//   warp 8           one thread loads by TMA: the query tiles once, K and V tiles round a ring
//   warp 9           one thread issues the products: S = Q K^T into tensor memory, and O += P V
//                    with P read from tensor memory, where it takes the place of S
//   warps 10, 11     look through the values of masked tiles (below)
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
// Every wait is bounded; one that gives up ends the block with NaN rows.

constexpr int kTcThreads = 384;
constexpr int kTcRows = 128;  // rows of a tile
constexpr int kTcKeys = 128;  // tokens of a key tile
constexpr int kTcLimit = 1 << 18;
constexpr float kLazy = 8.f;  // log2 of the growth of a maximum that is let pass

template <int DP>  // width rounded up to 64s
struct TcShape {
  static constexpr int kParts = DP / 64;                        // 128-byte wide parts of a row
  static constexpr int kPartBytes = 128 * 128;                  // 128 rows of one part
  static constexpr int kTileBytes = kParts * kPartBytes;
  static constexpr int kSlots = DP == 128 ? 4 : 8;              // ring of K and V tiles
  static constexpr int kBytes = (2 + kSlots) * kTileBytes + 1024;
};

struct TcLaunch {
  PromptLaunch p;
  CUtensorMap q, k, v;
};

struct TcBarriers {
  uint64_t full[8], empty[8];
  uint64_t q, s[2], p[2], o[2], look[2], looked[2], drain;  // look, looked: at most two tiles are masked
};

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
__device__ __forceinline__ void tc_store32(unsigned at, const unsigned* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::COW_W8(r, 0),
      COW_W8(r, 8), COW_W8(r, 16), COW_W8(r, 24), "r"(at)
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
template <int DT>
__device__ __forceinline__ bool any_nonfinite(unsigned w) {  // of the two 16-bit values
  constexpr unsigned kExp = DT == COW_BF16 ? 0x7f807f80u : 0x7c007c00u;
  const unsigned z = ~w & kExp;  // a half of zero: all exponent bits set
  return ((z - 0x00010001u) & ~z & 0x80008000u) != 0;
}

template <int DT, int DP>
__global__ void __launch_bounds__(kTcThreads, 1) cow_prompt_tc_kernel(const __grid_constant__ TcLaunch L) {
  using S = TcShape<DP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ TcBarriers bars;
  __shared__ Tile s_tile;
  __shared__ unsigned s_tmem;
  __shared__ int s_abort, s_bad;
  const PromptLaunch& P = L.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = P.group, tile_tokens = kTcRows / group, kv_head = blockIdx.x % P.kv_heads;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem;                          // tiles A and B
  uint8_t* s_ring = smem + 2 * S::kTileBytes;

  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (warp == 9) {
    if (lane == 0) {
      s_abort = s_bad = 0;
      for (int i = 0; i < S::kSlots; ++i) {
        mbar_init(&bars.full[i], 1);
        mbar_init(&bars.empty[i], 1);
      }
      mbar_init(&bars.q, 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars.s[i], 1);
        mbar_init(&bars.p[i], 4);
        mbar_init(&bars.o[i], 1);
        mbar_init(&bars.look[i], 1);
        mbar_init(&bars.looked[i], 2);
      }
      mbar_init(&bars.drain, 1);
    }
  } else if (warp == 10) {
    const Tile t = find_tile(P, 2 * tile_tokens, blockIdx.x / P.kv_heads);
    if (lane == 0) s_tile = t;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = s_tmem;
  const Tile t = s_tile;
  volatile int* abort = &s_abort;
  auto wait = [&](uint64_t* bar, unsigned parity) {
    if (*abort) return false;
    if (mbar_wait(bar, parity, kTcLimit)) return true;
    *abort = 1;
    return false;
  };

  // tokens and key tiles of A and B
  const int here_a = min(tile_tokens, t.count - t.first), here_b = max(min(tile_tokens, t.count - t.first - tile_tokens), 0);
  const int n_a = (t.first + here_a + kTcKeys - 1) / kTcKeys;
  const int n_b = here_b > 0 ? (t.first + tile_tokens + here_b + kTcKeys - 1) / kTcKeys : 0;
  const int n = max(n_a, n_b);
  const int masked_from = t.first / kTcKeys;  // key tiles from here on are not seen whole by every row

  if (t.count > 0) {
    if (warp == 8 && lane == 0) {
      // ---- loads
      mbar_arrive_expect_tx(&bars.q, (here_b > 0 ? 2 : 1) * S::kParts * 128 * group * tile_tokens);
      for (int x = 0; x < (here_b > 0 ? 2 : 1); ++x)
        for (int part = 0; part < S::kParts; ++part)
          tma_load(s_q + x * S::kTileBytes + part * S::kPartBytes, &L.q, 64 * part, kv_head * group,
                   t.begin + t.first + x * tile_tokens, &bars.q);
      int issued = 0;
      for (int i = 0; i < 2 * n; ++i) {  // K(0), V(0), K(1), ...
        const int slot = i % S::kSlots;
        if (i >= S::kSlots && !wait(&bars.empty[slot], (i / S::kSlots - 1) & 1)) break;
        mbar_arrive_expect_tx(&bars.full[slot], S::kTileBytes);
        for (int part = 0; part < S::kParts; ++part)
          tma_load(s_ring + slot * S::kTileBytes + part * S::kPartBytes, i & 1 ? &L.v : &L.k, 64 * part, kv_head,
                   t.begin + (i >> 1) * kTcKeys, &bars.full[slot]);
        issued = i + 1;
      }
      // nothing may still be on its way into shared memory when the block ends
      mbar_wait(&bars.q, 0, kTcLimit);
      for (int i = max(issued - S::kSlots, 0); i < issued; ++i) mbar_wait(&bars.full[i % S::kSlots], (i / S::kSlots) & 1, kTcLimit);
    } else if (warp == 9 && lane == 0) {
      // ---- products
      const int steps = (P.width + 15) / 16;
      constexpr unsigned kType = DT == COW_BF16 ? 1u : 0u;
      const unsigned base = (1u << 4) | (kType << 7) | (kType << 10) | ((128u >> 4) << 24);
      // S: 128 x 128, both operands contiguous along the width; a negative scale negates Q
      const unsigned idesc_s = base | ((128u >> 3) << 17) | (P.scale_log2 < 0.f ? 1u << 13 : 0u);
      // O: 128 x width, values contiguous along the output's columns
      const unsigned idesc_o = base | (1u << 16) | (static_cast<unsigned>(2 * steps) << 17);
      auto score = [&](int x, int j) {
        const unsigned q = smem_addr(s_q) + x * S::kTileBytes, k = smem_addr(s_ring) + (2 * j % S::kSlots) * S::kTileBytes;
        for (int i = 0; i < steps; ++i) {
          const unsigned off = (i / 4) * S::kPartBytes + (i % 4) * 32;
          tc_mma_ss(tmem + 128 * x, operand_at(q + off, 16), operand_at(k + off, 16), idesc_s, i > 0);
        }
      };
      auto output = [&](int x, int j) {
        const unsigned v = smem_addr(s_ring) + ((2 * j + 1) % S::kSlots) * S::kTileBytes;
        for (int i = 0; i < kTcKeys / 16; ++i)
          tc_mma_ts(tmem + 256 + 128 * x, tmem + 128 * x + 8 * i, operand_at(v + 2048 * i, S::kPartBytes), idesc_o, j > 0 || i > 0);
      };
      auto full = [&](int i) { return wait(&bars.full[i % S::kSlots], (i / S::kSlots) & 1); };
      bool ok = wait(&bars.q, 0) && full(0);
      if (ok) {
        tc_fence_after();
        score(0, 0);
        tc_commit(&bars.s[0]);
        if (n_b > 0) {
          score(1, 0);
          tc_commit(&bars.s[1]);
        }
        tc_commit(&bars.empty[0]);
      }
      for (int j = 0; ok && j < n; ++j) {
        ok = full(2 * j + 1);
        if (ok && j >= masked_from) mbar_arrive(&bars.look[j - masked_from]);
        ok = ok && (j + 1 >= n || full(2 * j + 2));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int nx = x ? n_b : n_a;
          if (!ok || j >= nx) continue;
          ok = wait(&bars.p[x], j & 1) && (j < masked_from || wait(&bars.looked[j - masked_from], 0));
          if (!ok) continue;
          tc_fence_after();
          output(x, j);
          if (j + 1 < nx) {
            score(x, j + 1);
            tc_commit(&bars.s[x]);
          } else {
            tc_commit(&bars.o[x]);
          }
        }
        if (ok) {
          tc_commit(&bars.empty[(2 * j + 1) % S::kSlots]);
          if (j + 1 < n) tc_commit(&bars.empty[(2 * j + 2) % S::kSlots]);
        }
      }
      if (!ok) {  // products in flight end before tensor memory is given back
        tc_commit(&bars.drain);
        mbar_wait(&bars.drain, 0, kTcLimit);
      }
    } else if (warp >= 10) {
      // ---- values of masked tiles
      for (int j = masked_from; j < n; ++j) {
        const int slot = (2 * j + 1) % S::kSlots;
        if (!__all_sync(kFull, wait(&bars.look[j - masked_from], 0) && wait(&bars.full[slot], ((2 * j + 1) / S::kSlots) & 1))) break;
        uint4* words = reinterpret_cast<uint4*>(s_ring + slot * S::kTileBytes);
        constexpr int kEach = S::kTileBytes / 16 / 64;
        bool bad = false;
#pragma unroll 8
        for (int i = 0; i < kEach; ++i) {
          const uint4 w = words[i * 64 + (warp - 10) * 32 + lane];
          bad |= any_nonfinite<DT>(w.x) | any_nonfinite<DT>(w.y) | any_nonfinite<DT>(w.z) | any_nonfinite<DT>(w.w);
        }
        if (bad) {
          constexpr unsigned kExp = DT == COW_BF16 ? 0x7f80u : 0x7c00u;
          s_bad = 1;
          for (int i = 0; i < kEach; ++i) {
            unsigned* w = reinterpret_cast<unsigned*>(words + i * 64 + (warp - 10) * 32 + lane);
            for (int u = 0; u < 4; ++u) {
              if ((w[u] & kExp) == kExp) w[u] &= 0xffff0000u;
              if (((w[u] >> 16) & kExp) == kExp) w[u] &= 0xffffu;
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.looked[j - masked_from]);
      }
    } else if (warp < 8) {
      // ---- softmax
      const int x = warp >> 2;
      const int nx = x ? n_b : n_a, here = x ? here_b : here_a;
      const int row = tid & 127, first = t.first + x * tile_tokens;
      const int query = first + row / group;  // its place in the sequence
      const unsigned lanes = tmem + (static_cast<unsigned>(warp & 3) << 21);  // this warp's 32 lanes
      const unsigned at_s = lanes + 128 * x, at_o = lanes + 256 + 128 * x;
      const float c = fabsf(P.scale_log2);
      float m = -INFINITY, l = 0.f;  // m: the maximum that P is relative to
      bool ok = true;
      for (int j = 0; j < nx; ++j) {
        ok = __all_sync(kFull, wait(&bars.s[x], j & 1));
        if (!ok) break;
        tc_fence_after();
        unsigned s[128];
        tc_load32(at_s, s);
        tc_load32(at_s + 32, s + 32);
        tc_load32(at_s + 64, s + 64);
        tc_load32(at_s + 96, s + 96);
        tc_wait_loads();
        if (j * kTcKeys + kTcKeys - 1 > first) {
          const int seen = query - j * kTcKeys;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i > seen) s[i] = 0xff800000u;
        }
        float big[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; ++i) big[i & 3] = fmaxf(big[i & 3], __uint_as_float(s[i]));
        const float now = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) * c;
        const bool grown = now > m + kLazy || m == -INFINITY;
        if (__any_sync(kFull, grown)) {
          const float next = grown ? fmaxf(now, m) : m;
          const float a = grown && next != -INFINITY ? exp2_fast(m - next) : 1.f;
          m = next;
          l *= a;
          if (j > 0) {
#pragma unroll 1
            for (int i = 0; i < P.width; i += 32) {
              unsigned o[32];
              tc_load32(at_o + i, o);
              tc_wait_loads();
#pragma unroll
              for (int u = 0; u < 32; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * a);
              tc_store32(at_o + i, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : m;  // all -inf so far: weights 0
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          unsigned p[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float e0 = exp2_fast(fmaf(__uint_as_float(s[64 * h + 2 * i]), c, -base));
            const float e1 = exp2_fast(fmaf(__uint_as_float(s[64 * h + 2 * i + 1]), c, -base));
            sum[0] += e0;
            sum[1] += e1;
            p[i] = pack2<DT>(e0, e1);
          }
          tc_store32(at_s + 32 * h, p);
        }
        l += sum[0] + sum[1];
        tc_wait_stores();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p[x]);
      }
      if (nx > 0) {
        ok = __all_sync(kFull, ok && wait(&bars.o[x], 0));
        tc_fence_after();
        const bool store = row / group < here;
        const float inv = ok ? 1.f / l : __int_as_float(0x7fc00000);
        uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(P.out) +
                                              (static_cast<int64_t>(t.begin + query) * P.heads +
                                               static_cast<int64_t>(kv_head) * group + row % group) * P.width);
#pragma unroll 1
        for (int i = 0; i < P.width; i += 32) {
          unsigned o[32];
          __syncwarp();
          tc_load32(at_o + i, o);
          tc_wait_loads();
          if (store && s_bad) {  // seen values that are not finite, taken out of the product above
            for (int j = masked_from * kTcKeys; j <= query; ++j) {
              const uint16_t* v = static_cast<const uint16_t*>(P.v) + (t.begin + j) * P.v_token + kv_head * P.v_head + i;
#pragma unroll
              for (int u = 0; u < 32; ++u) {
                if (i + u < P.width) {
                  const float f = DT == COW_BF16 ? __uint_as_float(static_cast<unsigned>(v[u]) << 16)
                                                 : __half2float(*reinterpret_cast<const __half*>(v + u));
                  if (!(fabsf(f) < INFINITY)) o[u] = __float_as_uint(__uint_as_float(o[u]) + f);
                }
              }
            }
          }
          if (store) {
#pragma unroll
            for (int u = 0; u < 32; u += 8) {
              if (i + u < P.width) {
                uint4 w;
                w.x = pack2<DT>(__uint_as_float(o[u]) * inv, __uint_as_float(o[u + 1]) * inv);
                w.y = pack2<DT>(__uint_as_float(o[u + 2]) * inv, __uint_as_float(o[u + 3]) * inv);
                w.z = pack2<DT>(__uint_as_float(o[u + 4]) * inv, __uint_as_float(o[u + 5]) * inv);
                w.w = pack2<DT>(__uint_as_float(o[u + 6]) * inv, __uint_as_float(o[u + 7]) * inv);
                out[(i + u) / 8] = w;
              }
            }
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
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
  if (!resident_blocks(reinterpret_cast<const void*>(cow_prompt_tc_kernel<DT, DP>), kTcThreads, TcShape<DP>::kBytes))
    return COW_ERR_CUDA;
  cow_prompt_tc_kernel<DT, DP><<<blocks, kTcThreads, TcShape<DP>::kBytes, stream>>>(L);
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
  if (P.dtype == COW_BF16)
    return P.width <= 64 ? launch_tc<COW_BF16, 64>(L, blocks, stream) : launch_tc<COW_BF16, 128>(L, blocks, stream);
  return P.width <= 64 ? launch_tc<COW_F16, 64>(L, blocks, stream) : launch_tc<COW_F16, 128>(L, blocks, stream);
}

template <int D>
int launch_f32(const PromptLaunch& P, unsigned blocks, cudaStream_t stream) {
  constexpr size_t kBytes = sizeof(float) * ((kRows + 2 * kKeys) * (D + 4) + kRows * (kKeys + 4));
  if (!resident_blocks(reinterpret_cast<const void*>(cow_prompt_f32_kernel<D>), kThreads, kBytes)) return COW_ERR_CUDA;
  cow_prompt_f32_kernel<D><<<blocks, kThreads, kBytes, stream>>>(P);
  return launch_status();
}

int prompt_f32(const PromptLaunch& P, cudaStream_t stream) {
  // every sequence adds at most one tile that is not full
  const int64_t tiles = P.tokens / (kRows / P.group) + (P.sequences < P.tokens ? P.sequences : P.tokens);
  const unsigned blocks = static_cast<unsigned>(tiles * P.kv_heads);
  if (P.width <= 32) return launch_f32<32>(P, blocks, stream);
  return P.width <= 64 ? launch_f32<64>(P, blocks, stream) : launch_f32<128>(P, blocks, stream);
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
                         int32_t dtype, float scale, void* out, void* stream) {
  if (!valid_dtype(dtype) || sequences < 0 || tokens < 0 || kv_heads < 1 || heads < 1 || heads % kv_heads || width < 1)
    return COW_ERR_INVALID;
  if (width % 8 || width > 128 || heads / kv_heads > kMaxGroup || tokens >= (int64_t{1} << 30) ||
      sequences >= (int64_t{1} << 30))
    return COW_ERR_UNSUPPORTED;
  if (sequences == 0 || tokens == 0) return COW_OK;
  if ((tokens / (kRows / (heads / kv_heads)) + (sequences < tokens ? sequences : tokens)) * kv_heads >= (int64_t{1} << 31))
    return COW_ERR_UNSUPPORTED;  // more blocks than one launch has
  if (!rows_ok(queries, query_token_stride, query_head_stride, dtype) ||
      !rows_ok(keys, key_token_stride, key_head_stride, dtype) ||
      !rows_ok(values, value_token_stride, value_head_stride, dtype) || !starts || !out || !aligned16(out))
    return COW_ERR_INVALID;
  PromptLaunch P{queries, keys, values, out, starts, query_token_stride, query_head_stride, key_token_stride,
                 key_head_stride, value_token_stride, value_head_stride, static_cast<int32_t>(sequences),
                 static_cast<int32_t>(tokens), heads, kv_heads, heads / kv_heads, width, dtype,
                 scale * 1.4426950408889634f};
  return dtype == COW_F32 ? prompt_f32(P, as_stream(stream)) : prompt_tc(P, as_stream(stream));
}

}  // extern "C"
