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
  int32_t sequences, tokens, heads, group, width, dtype;
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
__global__ void __launch_bounds__(kThreads) cow_prompt_kernel(const __grid_constant__ PromptLaunch P) {
  constexpr int kStride = D + 4;
  constexpr int kCols = D / 16;
  extern __shared__ __align__(16) float smem_f[];
  float* s_q = smem_f;                     // [kRows][kStride]
  float* s_k = s_q + kRows * kStride;      // [kKeys][kStride]
  float* s_v = s_k + kKeys * kStride;      // [kKeys][kStride]
  float* s_p = s_v + kKeys * kStride;      // [kRows][kKeys + 4]
  __shared__ Tile s_tile;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int group = P.group, tile_tokens = kRows / group, kv_head = blockIdx.y, W = P.width;
  if (tid < 32) {
    const Tile t = find_tile(P, tile_tokens, blockIdx.x);
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
  if (width % 8 || width > 128 || heads / kv_heads > kMaxGroup || kv_heads > 65535 || tokens >= (int64_t{1} << 30) ||
      sequences >= (int64_t{1} << 30))
    return COW_ERR_UNSUPPORTED;
  if (sequences == 0 || tokens == 0) return COW_OK;
  if (!rows_ok(queries, query_token_stride, query_head_stride, dtype) ||
      !rows_ok(keys, key_token_stride, key_head_stride, dtype) ||
      !rows_ok(values, value_token_stride, value_head_stride, dtype) || !starts || !out || !aligned16(out))
    return COW_ERR_INVALID;
  PromptLaunch P{queries, keys, values, out, starts, query_token_stride, query_head_stride, key_token_stride,
                 key_head_stride, value_token_stride, value_head_stride, static_cast<int32_t>(sequences),
                 static_cast<int32_t>(tokens), heads, heads / kv_heads, width, dtype, scale * 1.4426950408889634f};
  const int tile_tokens = kRows / P.group;
  const void* fn;
  int D = width <= 32 ? 32 : width <= 64 ? 64 : 128;
  fn = D == 32 ? reinterpret_cast<const void*>(cow_prompt_kernel<32>)
               : D == 64 ? reinterpret_cast<const void*>(cow_prompt_kernel<64>)
                         : reinterpret_cast<const void*>(cow_prompt_kernel<128>);
  const size_t smem = sizeof(float) * ((kRows + 2 * kKeys) * (D + 4) + kRows * (kKeys + 4));
  if (!resident_blocks(fn, kThreads, smem)) return COW_ERR_CUDA;
  // every sequence adds at most one tile that is not full
  const int64_t tiles = tokens / tile_tokens + (sequences < tokens ? sequences : tokens);
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(kv_heads));
  if (D == 32) cow_prompt_kernel<32><<<grid, kThreads, smem, as_stream(stream)>>>(P);
  else if (D == 64) cow_prompt_kernel<64><<<grid, kThreads, smem, as_stream(stream)>>>(P);
  else cow_prompt_kernel<128><<<grid, kThreads, smem, as_stream(stream)>>>(P);
  return launch_status();
}

}  // extern "C"
