// cow_kv8.cu -- the paged K/V cache held in 8 bits: store, read back, attend.
//
// A page holds 64 tokens of one key/value head as e4m3 codes with one scale for its keys and
// one for its values.  Scales are powers of two: a code keeps the same four significant bits
// whatever the scale's mantissa would be, so a finer scale gains nothing, while x / scale
// is exact before its one rounding, and when a later token of the page needs a larger scale,
// the codes already there move to it exactly (but for those that become subnormal).
// Keys lie [token][width]; values lie transposed, [width][token], so that one lane's 16-byte
// word of either is the operand of a matrix instruction without any exchange.

#include <cuda_fp8.h>

#include "cow_common.cuh"

namespace {

constexpr int kPage = COW_PAGE_TOKENS;
constexpr int kStoreThreads = 128;
constexpr int kStoreWarps = kStoreThreads / 32;
constexpr int kLeastExponent = -64;

// --------------------------------------------------------------------------
// codes
// --------------------------------------------------------------------------

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // e in [-126, 127]

// Smallest e >= kLeastExponent with most <= 448 * 2^e; 448 = 1.75 * 2^8, so only the
// exponent of `most` and whether its mantissa is above 1.75 count.  most is finite, >= 0.
__device__ __forceinline__ int scale_exponent(float most) {
  const int bits = __float_as_int(most);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return max(e, kLeastExponent);
}
__device__ __forceinline__ int exponent_of(float scale) { return (__float_as_int(scale) >> 23) - 127; }

__device__ __forceinline__ unsigned encode2(float a, float b) {  // a in the low byte; to nearest even, saturating
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ unsigned encode4(float a, float b, float c, float d) {
  return encode2(a, b) | (encode2(c, d) << 16);
}
__device__ __forceinline__ float2 decode2(unsigned codes) {  // the two low bytes
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ unsigned recode4(unsigned codes, float ratio) {
  const float2 a = decode2(codes), b = decode2(codes >> 16);
  return encode4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}

// 16 bytes of a tensor as floats
template <int DT>
struct Vec16;
template <>
struct Vec16<COW_F32> {
  static constexpr int kElems = 4;
  static __device__ __forceinline__ void get(uint4 u, float* x) {
    x[0] = __uint_as_float(u.x);
    x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z);
    x[3] = __uint_as_float(u.w);
  }
};
template <>
struct Vec16<COW_BF16> {
  static constexpr int kElems = 8;
  static __device__ __forceinline__ void get(uint4 u, float* x) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct Vec16<COW_F16> {
  static constexpr int kElems = 8;
  static __device__ __forceinline__ void get(uint4 u, float* x) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};

template <int DT>
__device__ __forceinline__ float most_of(uint4 u, float most) {
  float x[Vec16<DT>::kElems];
  Vec16<DT>::get(u, x);
#pragma unroll
  for (int i = 0; i < Vec16<DT>::kElems; ++i) {
    const float a = fabsf(x[i]);
    if (a < INFINITY) most = fmaxf(most, a);  // infinities and NaN do not set a scale
  }
  return most;
}

// --------------------------------------------------------------------------
// store
// --------------------------------------------------------------------------
//
// One block per (page piece, head) of the plan: the piece's tokens of keys, then of values,
// are read once into registers, their largest magnitude gives the scale, and the codes are
// written.  Keys: a thread's 16 bytes are neighbours of the next thread's.  Values: a lane
// reads one 16-byte word of each of four neighbouring tokens and so holds whole 32-bit words
// of four codes of the transposed page; two lanes share a 32-byte sector.
// Bound: memory, (element size + 1) bytes for each element of keys and values.

struct StoreLaunch {
  uint8_t* codes[2];  // keys, values: this layer's pages
  float* scales[2];
  const char* x[2];
  int64_t token_stride[2], head_stride[2];  // bytes
  const int32_t* plan;
  int32_t kv_heads, pages;
};

__device__ __forceinline__ float block_most(float most, float* s_red, int lane, int warp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(kFull, most, o));
  __syncthreads();  // the previous use of s_red is over
  if (lane == 0) s_red[warp] = most;
  __syncthreads();
  most = s_red[0];
#pragma unroll
  for (int w = 1; w < kStoreWarps; ++w) most = fmaxf(most, s_red[w]);
  return most;
}

template <int DT, int D>
__global__ void __launch_bounds__(kStoreThreads) cow_kv8_store_kernel(const __grid_constant__ StoreLaunch P) {
  constexpr int E = Vec16<DT>::kElems;
  constexpr int kVecs = D / E;                                          // 16-byte words per token
  constexpr int kKeyVecs = (kPage * kVecs + kStoreThreads - 1) / kStoreThreads;
  constexpr int kGroups = D / (2 * E);                                  // pairs of words per token
  constexpr int kValueGroups = (kGroups + kStoreWarps - 1) / kStoreWarps;
  __shared__ float s_red[kStoreWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y;
  if (static_cast<int>(blockIdx.x) >= P.plan[0]) return;
  const int4 piece = reinterpret_cast<const int4*>(P.plan + 4)[blockIdx.x];
  const int first = piece.x, tokens = piece.y, page = piece.z, offset = piece.w;
  if (page < 0 || page >= P.pages) return;
  const int64_t tile = static_cast<int64_t>(page) * P.kv_heads + head;

  // ---- keys
  {
    const char* src = P.x[0] + first * P.token_stride[0] + head * P.head_stride[0];
    uint8_t* dst = P.codes[0] + tile * (kPage * D);
    uint4 w[kKeyVecs];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kKeyVecs; ++i) {
      const int v = tid + i * kStoreThreads;
      if (v < tokens * kVecs)
        w[i] = __ldg(reinterpret_cast<const uint4*>(src + (v / kVecs) * P.token_stride[0]) + v % kVecs);
    }
#pragma unroll
    for (int i = 0; i < kKeyVecs; ++i)
      if (tid + i * kStoreThreads < tokens * kVecs) most = most_of<DT>(w[i], most);
    int e = scale_exponent(block_most(most, s_red, lane, warp));
    if (offset > 0) {
      const int old = exponent_of(P.scales[0][tile]);
      e = max(e, old);
      if (e > old) {
        const float ratio = e - old > 126 ? 0.f : pow2(old - e);
        for (int i = tid; i < offset * D / 4; i += kStoreThreads) {
          unsigned* word = reinterpret_cast<unsigned*>(dst) + i;
          *word = recode4(*word, ratio);
        }
      }
    }
    const float inv = pow2(-e);
#pragma unroll
    for (int i = 0; i < kKeyVecs; ++i) {
      const int v = tid + i * kStoreThreads;
      if (v < tokens * kVecs) {
        float x[E];
        Vec16<DT>::get(w[i], x);
        unsigned* out = reinterpret_cast<unsigned*>(dst + offset * D + v * E);
#pragma unroll
        for (int j = 0; j < E; j += 4) out[j / 4] = encode4(x[j] * inv, x[j + 1] * inv, x[j + 2] * inv, x[j + 3] * inv);
      }
    }
    __syncthreads();  // every thread has read the old scale
    if (tid == 0) P.scales[0][tile] = pow2(e);
  }

  // ---- values
  {
    const char* src = P.x[1] + head * P.head_stride[1];
    uint8_t* dst = P.codes[1] + tile * (kPage * D);
    const int t0 = (lane >> 1) * 4;  // this lane's four tokens of the page
    uint4 w[kValueGroups][4];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kValueGroups; ++i) {
      const int g = warp + i * kStoreWarps;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + j - offset;
        w[i][j] = make_uint4(0, 0, 0, 0);
        if (g < kGroups && t >= 0 && t < tokens)
          w[i][j] = __ldg(reinterpret_cast<const uint4*>(src + (first + t) * P.token_stride[1]) + 2 * g + (lane & 1));
      }
    }
#pragma unroll
    for (int i = 0; i < kValueGroups; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) most = most_of<DT>(w[i][j], most);
    int e = scale_exponent(block_most(most, s_red, lane, warp));
    if (offset > 0) {
      const int old = exponent_of(P.scales[1][tile]);
      e = max(e, old);
      if (e > old) {
        const float ratio = e - old > 126 ? 0.f : pow2(old - e);
        const int words = (offset + 3) / 4;  // the last may hold bytes past the old tokens: written after the barrier
        for (int i = tid; i < D * words; i += kStoreThreads) {
          unsigned* word = reinterpret_cast<unsigned*>(dst + (i / words) * kPage) + i % words;
          *word = recode4(*word, ratio);
        }
      }
    }
    __syncthreads();
    const float inv = pow2(-e);
#pragma unroll
    for (int i = 0; i < kValueGroups; ++i) {
      const int g = warp + i * kStoreWarps;
      const int have = min(t0 + 4, offset + tokens) - max(t0, offset);
      if (g < kGroups && have > 0) {
        float x[4][E];
#pragma unroll
        for (int j = 0; j < 4; ++j) Vec16<DT>::get(w[i][j], x[j]);
#pragma unroll
        for (int d = 0; d < E; ++d) {
          const unsigned codes = encode4(x[0][d] * inv, x[1][d] * inv, x[2][d] * inv, x[3][d] * inv);
          uint8_t* out = dst + ((2 * g + (lane & 1)) * E + d) * kPage + t0;
          if (have == 4) {
            *reinterpret_cast<unsigned*>(out) = codes;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (t0 + j >= offset && t0 + j < offset + tokens) out[j] = static_cast<uint8_t>(codes >> (8 * j));
          }
        }
      }
    }
    if (tid == 0) P.scales[1][tile] = pow2(e);
  }
}

// --------------------------------------------------------------------------
// read
// --------------------------------------------------------------------------
//
// One block per (32 slots, head).  Keys: a warp takes a slot, each lane four codes of its row.
// Values: a lane takes a slot and the block walks the width, so neighbouring slots of a page
// share each 32-byte sector; the codes cross shared memory to leave as rows.

struct ReadLaunch {
  const uint8_t* codes[2];
  const float* scales[2];
  char* out[2];
  const int32_t* slots;
  int64_t count;
  int32_t kv_heads, pages, width, dtype;
};

constexpr int kReadSlots = 32;

__global__ void __launch_bounds__(kStoreThreads) cow_kv8_read_kernel(const __grid_constant__ ReadLaunch P) {
  __shared__ uint8_t s_codes[kReadSlots][128 + 4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = P.width, head = blockIdx.y;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kReadSlots;
  const int here = static_cast<int>(min(static_cast<int64_t>(kReadSlots), P.count - base));
  const int limit = P.pages * kPage;
  // values: into shared memory, transposed
  {
    const int slot = lane < here ? P.slots[base + lane] : -1;
    const bool ok = slot >= 0 && slot < limit;
    const uint8_t* src = P.codes[1] + (static_cast<int64_t>(ok ? slot / kPage : 0) * P.kv_heads + head) * (kPage * D) +
                         (ok ? slot % kPage : 0);
    for (int d = warp; d < D; d += kStoreWarps) s_codes[lane][d] = ok ? src[d * kPage] : 0;
  }
  __syncthreads();
  for (int i = warp; i < here; i += kStoreWarps) {
    const int slot = P.slots[base + i];
    const bool ok = slot >= 0 && slot < limit;
    const int64_t tile = static_cast<int64_t>(ok ? slot / kPage : 0) * P.kv_heads + head;
    const int64_t row = (base + i) * P.kv_heads + head;
    if (4 * lane < D) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        unsigned codes = 0;
        float scale = 0.f;
        if (ok) {
          scale = P.scales[which][tile];
          codes = which ? *reinterpret_cast<const unsigned*>(&s_codes[i][4 * lane])
                        : *reinterpret_cast<const unsigned*>(P.codes[0] + tile * (kPage * D) + (slot % kPage) * D + 4 * lane);
        }
        const float2 a = decode2(codes), b = decode2(codes >> 16);
        st4_rt(P.out[which], row * D + 4 * lane, make_float4(a.x * scale, a.y * scale, b.x * scale, b.y * scale), P.dtype);
      }
    }
  }
}

// --------------------------------------------------------------------------
// attend
// --------------------------------------------------------------------------
//
// One query token per request, s_j = scale * ks * (q . k_j), o = sum_j softmax(s)_j vs v_j with
// the code's k_j, v_j and the page's ks, vs.  Bound: memory, 2 * width bytes for each cached token
// and key head, everything else is small.  So:
// * the pages of all requests and heads form one list, cut into equal runs, one for each
//   resident block, whatever the requests' lengths; a (request, head) pair that several blocks share
//   is joined, in the order of its pages, by the block that finishes last;
// * within a run a warp takes every fourth page; its K and V codes come by 16-byte asynchronous
//   copies, the next page's keys while this page's values are used, and every lane reads back only
//   what it copied itself, so nothing waits for another lane;
// * e4m3 is exact in f16, so both products run on m16n8k16 with f16 operands and f32 sums: pages are
//   the 16-row operand (tokens, then width), the group's query heads the 8 columns, eight heads
//   to a block.  The tcgen05 form would need the codes widened in shared memory first; here they
//   go from the 16-byte words to operands in registers, and at 4 heads to a key the whole
//   contraction is 1/10 of what this instruction sustains at the memory's rate.
//   Queries are scaled per head by a power of two into f16's range; f32 ones are
//   held as two f16 parts (22 bits), and so are their probabilities.
// * running maximum, sum and output of the softmax stay in f32 registers; value scales,
//   powers of two, ride on the factor that rescales the output when the maximum moves.

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = 32 * kAttendWarps;
constexpr int kAttendHeads = 8;   // query heads of one block: the matrix instruction's columns
constexpr float kProbShift = 8.f;  // probabilities are held times 2^8: more of f16's range below the largest

struct AttendLaunch {
  const uint8_t* key_codes;
  const uint8_t* value_codes;
  const float* key_scales;
  const float* value_scales;
  const int32_t* tables;
  const int32_t* lengths;
  const char* q;
  char* out;
  float* partials;  // [2 * blocks][8 * (width + 2)]
  unsigned* arrived;  // [requests * pairs]
  int32_t* status;
  int64_t q_request_stride, q_head_stride;  // elements
  int64_t max_blocks;
  int32_t requests, kv_heads, heads, group, chunks, pages, dtype;
  float scale_log2;  // scale * log2(e)
};

__device__ __forceinline__ unsigned widen2(unsigned short codes) {
  unsigned h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(codes));
  return h;
}
__device__ __forceinline__ unsigned lo2(unsigned w) { return widen2(static_cast<unsigned short>(w & 0xffffu)); }
__device__ __forceinline__ unsigned hi2(unsigned w) { return widen2(static_cast<unsigned short>(w >> 16)); }

__device__ __forceinline__ void mma_f16(float* c, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                        unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
// what f16 leaves of a and b
__device__ __forceinline__ unsigned pack_rest2(float a, float b, unsigned packed) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&packed));
  return pack_half2(a - h.x, b - h.y);
}

__device__ __forceinline__ void copy16(unsigned smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void copy8(unsigned smem, const void* gmem) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Lane (g = lane / 4, c = lane % 4) of a warp holds of a 64-token page, for the four 16-row steps s:
//   keys:   tokens 16 (g/2) + 4 s + g%2 and that + 2 (rows g and g + 8 of step s), of each the 16 bytes
//           64 h + 16 c of every whole 64-byte part h of the row and 8 bytes 64 H + 8 c of a last half one;
//   values: rows 8 i + g of the width, of each the 16 tokens 16 c .. 16 c + 15.
// Word q of a key chunk is width 4 q .. 4 q + 3 from its start: operand columns 2c, 2c+1 and 2c+8, 2c+9 of one
// k16 step; word s of a value chunk is tokens 16 c + 4 s ..+3, the same columns of step s.  The order of
// a contraction's terms is free, so queries and probabilities only have to follow the same order.
template <int D>
struct PageShape {
  static constexpr int kWhole = D / 64;                 // 64-byte parts of a key row
  static constexpr int kHalf = (D % 64) / 32;           // a last 32-byte part
  static constexpr int kKeySteps = D / 16;              // k16 steps of q . k
  static constexpr int kValueRows = D / 8;              // value rows per lane
  static constexpr int kBytes = kPage * D;
};

template <int D>
__device__ __forceinline__ void copy_keys(unsigned smem, const uint8_t* tile, int lane) {
  using S = PageShape<D>;
  const int g = lane >> 2, c = lane & 3;
  const uint8_t* src = tile + ((g >> 1) * 16 + (g & 1)) * D;
#pragma unroll
  for (int r = 0; r < 8; ++r) {  // r = 2 s + half
    const uint8_t* row = src + 2 * r * D;
#pragma unroll
    for (int h = 0; h < S::kWhole; ++h) copy16(smem + ((r * S::kWhole + h) * 32 + lane) * 16, row + 64 * h + 16 * c);
    if constexpr (S::kHalf)
      copy8(smem + S::kWhole * 64 * kPage + (r * 32 + lane) * 8, row + 64 * S::kWhole + 8 * c);
  }
}
template <int D>
__device__ __forceinline__ void copy_values(unsigned smem, const uint8_t* tile, int lane) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int i = 0; i < PageShape<D>::kValueRows; ++i) copy16(smem + (i * 32 + lane) * 16, tile + (8 * i + g) * kPage + 16 * c);
}

struct Run {  // the part of one (request, head chunk)'s pages that a block has
  int request, pair, first, last, pages;  // pages first..last-1 of `pages`
};

template <int D, bool kSplit>
__global__ void __launch_bounds__(kAttendThreads) cow_kv8_attend_kernel(const __grid_constant__ AttendLaunch P) {
  using S = PageShape<D>;
  constexpr int kRow = D + 2;  // a partial's row: output, maximum, sum
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  uint8_t* s_keys = smem + warp * 2 * S::kBytes;
  uint8_t* s_values = s_keys + S::kBytes;
  int* s_prefix = reinterpret_cast<int*>(smem + kAttendWarps * 2 * S::kBytes);  // [requests + 1] pages before
  __shared__ int s_scan[kAttendWarps];
  __shared__ unsigned s_last;
  const int R = P.requests, pairs = P.kv_heads * P.chunks, G = gridDim.x;

  // pages of each request, and before it
  const int per = (R + kAttendThreads - 1) / kAttendThreads;
  const int most = static_cast<int>(P.max_blocks) * kPage;
  int sum = 0;
  for (int b = tid * per; b < min(R, (tid + 1) * per); ++b)
    sum += (min(max(P.lengths[b], 0), most) + kPage - 1) / kPage;
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(kFull, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) s_scan[warp] = inc;
  __syncthreads();
  int at = inc - sum, all = 0;
  for (int w = 0; w < kAttendWarps; ++w) {
    if (w < warp) at += s_scan[w];
    all += s_scan[w];
  }
  for (int b = tid * per; b < min(R, (tid + 1) * per); ++b) {
    s_prefix[b] = at;
    at += (min(max(P.lengths[b], 0), most) + kPage - 1) / kPage;
  }
  if (tid == 0) s_prefix[R] = all;
  __syncthreads();

  // a request without tokens: zeros
  for (int b = blockIdx.x; b < R; b += G) {
    if (s_prefix[b + 1] == s_prefix[b])
      for (int i = tid; i < P.heads * D / 4; i += kAttendThreads)
        st4_rt(P.out, static_cast<int64_t>(b) * P.heads * D + 4 * i, make_float4(0.f, 0.f, 0.f, 0.f), P.dtype);
  }

  // this block's run of the list (request, pair, page); at least a page for each warp
  const int64_t total = static_cast<int64_t>(all) * pairs;
  const int64_t share = max((total + G - 1) / G, static_cast<int64_t>(kAttendWarps));
  int64_t here = blockIdx.x * share;
  const int64_t end = min(here + share, total);

  while (here < end) {
    // which request, pair and page the run stands at
    int lo = 0, hi = R;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<int64_t>(s_prefix[mid]) * pairs <= here) lo = mid; else hi = mid;
    }
    const int b = lo, np = s_prefix[b + 1] - s_prefix[b];
    const int64_t before = static_cast<int64_t>(s_prefix[b]) * pairs;
    const int pair = static_cast<int>((here - before) / np);
    const int64_t pair_begin = before + static_cast<int64_t>(pair) * np;
    const int p_first = static_cast<int>(here - pair_begin);
    const int p_last = static_cast<int>(min(static_cast<int64_t>(np), end - pair_begin));
    here = pair_begin + p_last;
    const int kv_head = pair / P.chunks, chunk = pair % P.chunks;
    const int length = min(P.lengths[b], most);
    const int head0 = kv_head * P.group + chunk * kAttendHeads;
    const int heads_here = min(kAttendHeads, P.group - chunk * kAttendHeads);
    const int32_t* table = P.tables + b * P.max_blocks;

    auto tile_of = [&](int p) {
      int page = table[p];
      if (page < 0 || page >= P.pages) {
        if (lane == 0) atomicOr(P.status, COW_ST_ROW_RANGE);
        page = 0;
      }
      return static_cast<int64_t>(page) * P.kv_heads + kv_head;
    };

    int p = p_first + warp;
    int64_t tile = 0;
    float ks = 0.f, vs = 0.f;
    if (p < p_last) {
      tile = tile_of(p);
      copy_keys<D>(smem_addr(s_keys), P.key_codes + tile * S::kBytes, lane);
      copies_commit();
      copy_values<D>(smem_addr(s_values), P.value_codes + tile * S::kBytes, lane);
      copies_commit();
      ks = P.key_scales[tile];
      vs = P.value_scales[tile];
    }

    // the query of column g as operand columns, scaled so that its largest element is in [2^14, 2^15)
    unsigned qa[S::kKeySteps][2], qb[kSplit ? S::kKeySteps : 1][2];
    float unscale;
    {
      float x[S::kKeySteps][4];
      float big = 0.f;
      const bool there = g < heads_here;
      const int64_t row = b * P.q_request_stride + static_cast<int64_t>(head0 + (there ? g : 0)) * P.q_head_stride;
#pragma unroll
      for (int k = 0; k < S::kKeySteps; ++k) {
        const int h = k / 4;
        const int d = h < S::kWhole ? 64 * h + 16 * c + 4 * (k % 4) : 64 * S::kWhole + 8 * c + 4 * (k % 2);
        const float4 v = ld4_rt(P.q, row + d, P.dtype);
        x[k][0] = there ? v.x : 0.f;
        x[k][1] = there ? v.y : 0.f;
        x[k][2] = there ? v.z : 0.f;
        x[k][3] = there ? v.w : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (fabsf(x[k][i]) < INFINITY) big = fmaxf(big, fabsf(x[k][i]));
      }
      big = fmaxf(big, __shfl_xor_sync(kFull, big, 1));
      big = fmaxf(big, __shfl_xor_sync(kFull, big, 2));
      const int e = min(max(14 - exponent_of(big), -100), 100);
      const float up = pow2(e);
      unscale = pow2(-e);
#pragma unroll
      for (int k = 0; k < S::kKeySteps; ++k) {
        qa[k][0] = pack_half2(x[k][0] * up, x[k][1] * up);
        qa[k][1] = pack_half2(x[k][2] * up, x[k][3] * up);
        if constexpr (kSplit) {
          qb[k][0] = pack_rest2(x[k][0] * up, x[k][1] * up, qa[k][0]);
          qb[k][1] = pack_rest2(x[k][2] * up, x[k][3] * up, qa[k][1]);
        }
      }
    }
    // this lane's score columns are heads 2c and 2c + 1
    const float f0 = __shfl_sync(kFull, unscale, 8 * c) * P.scale_log2;
    const float f1 = __shfl_sync(kFull, unscale, 8 * c + 4) * P.scale_log2;

    float o[D / 16][4];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    int ve = 0;  // the output is held in units of 2^ve

    for (; p < p_last; p += kAttendWarps) {
      const int next = p + kAttendWarps;
      const bool more = next < p_last;
      int64_t next_tile = 0;
      if (more) next_tile = tile_of(next);

      copies_wait<1>();  // the keys are here
      float s[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
        const uint8_t* chunk0 = s_keys + lane * 16;
#pragma unroll
        for (int h = 0; h < S::kWhole; ++h) {
          const uint4 a = *reinterpret_cast<const uint4*>(chunk0 + ((2 * t) * S::kWhole + h) * 512);
          const uint4 z = *reinterpret_cast<const uint4*>(chunk0 + ((2 * t + 1) * S::kWhole + h) * 512);
          const unsigned aw[4] = {a.x, a.y, a.z, a.w}, zw[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const unsigned a0 = lo2(aw[q]), a1 = lo2(zw[q]), a2 = hi2(aw[q]), a3 = hi2(zw[q]);
            mma_f16(s[t], a0, a1, a2, a3, qa[4 * h + q][0], qa[4 * h + q][1]);
            if constexpr (kSplit) mma_f16(s[t], a0, a1, a2, a3, qb[4 * h + q][0], qb[4 * h + q][1]);
          }
        }
        if constexpr (S::kHalf) {
          const uint8_t* chunk1 = s_keys + S::kWhole * 64 * kPage + lane * 8;
          const uint2 a = *reinterpret_cast<const uint2*>(chunk1 + (2 * t) * 256);
          const uint2 z = *reinterpret_cast<const uint2*>(chunk1 + (2 * t + 1) * 256);
          const unsigned aw[2] = {a.x, a.y}, zw[2] = {z.x, z.y};
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            constexpr int k0 = 4 * S::kWhole;
            const unsigned a0 = lo2(aw[q]), a1 = lo2(zw[q]), a2 = hi2(aw[q]), a3 = hi2(zw[q]);
            mma_f16(s[t], a0, a1, a2, a3, qa[k0 + q][0], qa[k0 + q][1]);
            if constexpr (kSplit) mma_f16(s[t], a0, a1, a2, a3, qb[k0 + q][0], qb[k0 + q][1]);
          }
        }
      }
      if (more) copy_keys<D>(smem_addr(s_keys), P.key_codes + next_tile * S::kBytes, lane);
      copies_commit();

      // scores, the page's maximum, probabilities
      const int left = length - p * kPage;  // tokens of this page, if below 64
      const float fk0 = f0 * ks, fk1 = f1 * ks;
      float big0 = -INFINITY, big1 = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int token = (g >> 1) * 16 + 4 * t + (g & 1);
        s[t][0] = token < left ? s[t][0] * fk0 : -INFINITY;
        s[t][1] = token < left ? s[t][1] * fk1 : -INFINITY;
        s[t][2] = token + 2 < left ? s[t][2] * fk0 : -INFINITY;
        s[t][3] = token + 2 < left ? s[t][3] * fk1 : -INFINITY;
        big0 = fmaxf(big0, fmaxf(s[t][0], s[t][2]));
        big1 = fmaxf(big1, fmaxf(s[t][1], s[t][3]));
      }
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        big0 = fmaxf(big0, __shfl_xor_sync(kFull, big0, x));
        big1 = fmaxf(big1, __shfl_xor_sync(kFull, big1, x));
      }
      const float n0 = fmaxf(m0, big0), n1 = fmaxf(m1, big1);
      // where every score so far is -inf, exponents are taken from 0: probabilities 0, no NaN
      const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
      float a0 = exp2_fast(m0 - b0), a1 = exp2_fast(m1 - b1);
      m0 = n0;
      m1 = n1;
      l0 *= a0;
      l1 *= a1;
      // The output follows the page's value scale; a page 2^64 below the others keeps theirs and
      // its probabilities shrink instead, so no factor overflows.
      if (p == p_first + warp) ve = exponent_of(vs);
      int step = ve - exponent_of(vs);
      float shrink = 1.f;
      if (step > 64) {
        shrink = pow2(max(-step, -126));
        step = 0;
      }
      ve -= step;
      const float follow = step < -126 ? 0.f : pow2(step);
      a0 *= follow;
      a1 *= follow;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        o[i][0] *= a0;
        o[i][1] *= a1;
        o[i][2] *= a0;
        o[i][3] *= a1;
      }
      unsigned pa[4][2], pb[kSplit ? 4 : 1][2];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float e0 = exp2_fast(s[t][0] - b0 + kProbShift), e1 = exp2_fast(s[t][1] - b1 + kProbShift);
        const float e2 = exp2_fast(s[t][2] - b0 + kProbShift), e3 = exp2_fast(s[t][3] - b1 + kProbShift);
        l0 += e0 + e2;
        l1 += e1 + e3;
        const unsigned u0 = pack_half2(e0 * shrink, e1 * shrink), u1 = pack_half2(e2 * shrink, e3 * shrink);
        pa[t][0] = transpose8x8(u0);
        pa[t][1] = transpose8x8(u1);
        if constexpr (kSplit) {
          pb[t][0] = transpose8x8(pack_rest2(e0 * shrink, e1 * shrink, u0));
          pb[t][1] = transpose8x8(pack_rest2(e2 * shrink, e3 * shrink, u1));
        }
      }

      copies_wait<1>();  // the values are here
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        uint4 a = *reinterpret_cast<const uint4*>(s_values + ((2 * i) * 32 + lane) * 16);
        uint4 z = *reinterpret_cast<const uint4*>(s_values + ((2 * i + 1) * 32 + lane) * 16);
        unsigned aw[4] = {a.x, a.y, a.z, a.w}, zw[4] = {z.x, z.y, z.z, z.w};
        if (left < kPage) {  // codes past the last token may be anything, NaN among them: 0 * NaN is not 0
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int keep = min(max(left - (16 * c + 4 * t), 0), 4);
            const unsigned mask = keep == 4 ? 0xffffffffu : (1u << (8 * keep)) - 1u;
            aw[t] &= mask;
            zw[t] &= mask;
          }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const unsigned v0 = lo2(aw[t]), v1 = lo2(zw[t]), v2 = hi2(aw[t]), v3 = hi2(zw[t]);
          mma_f16(o[i], v0, v1, v2, v3, pa[t][0], pa[t][1]);
          if constexpr (kSplit) mma_f16(o[i], v0, v1, v2, v3, pb[t][0], pb[t][1]);
        }
      }
      if (more) {
        copy_values<D>(smem_addr(s_values), P.value_codes + next_tile * S::kBytes, lane);
        ks = P.key_scales[next_tile];
        vs = P.value_scales[next_tile];
      }
      copies_commit();
    }
    copies_wait<0>();
    // the sums over this warp's lanes
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l0 += __shfl_xor_sync(kFull, l0, x);
      l1 += __shfl_xor_sync(kFull, l1, x);
    }

    // ---- the block's four warps meet in shared memory (their pages are used up)
    __syncwarp();
    float* mine = reinterpret_cast<float*>(s_keys);  // [8][D + 2]
    const float unit = pow2(min(max(ve, -126), 127));
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      mine[(2 * c) * kRow + 16 * i + g] = o[i][0] * unit;
      mine[(2 * c + 1) * kRow + 16 * i + g] = o[i][1] * unit;
      mine[(2 * c) * kRow + 16 * i + g + 8] = o[i][2] * unit;
      mine[(2 * c + 1) * kRow + 16 * i + g + 8] = o[i][3] * unit;
    }
    if (g == 0) {
      mine[(2 * c) * kRow + D] = m0;
      mine[(2 * c) * kRow + D + 1] = l0;
      mine[(2 * c + 1) * kRow + D] = m1;
      mine[(2 * c + 1) * kRow + D + 1] = l1;
    }
    __syncthreads();
    const bool whole = p_first == 0 && p_last == np;
    const int64_t pair_end = pair_begin + np;
    const int64_t first_block = pair_begin / share;
    const int sharers = static_cast<int>((pair_end - 1) / share - first_block) + 1;
    float* partial = P.partials + (2 * static_cast<int64_t>(blockIdx.x) + (p_first == 0 ? 1 : 0)) * (kAttendHeads * kRow);
    for (int i = tid; i < heads_here * D; i += kAttendThreads) {
      const int h = i / D, d = i % D;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) m = fmaxf(m, reinterpret_cast<float*>(smem + w * 2 * S::kBytes)[h * kRow + D]);
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f, v = 0.f;
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) {
        const float* r = reinterpret_cast<float*>(smem + w * 2 * S::kBytes) + h * kRow;
        const float f = exp2_fast(r[D] - base);
        l = fmaf(f, r[D + 1], l);
        v = fmaf(f, r[d], v);
      }
      if (whole) {
        const float y = v / l;
        const int64_t at_out = (static_cast<int64_t>(b) * P.heads + head0 + h) * D + d;
        if (P.dtype == COW_F32) reinterpret_cast<float*>(P.out)[at_out] = y;
        else if (P.dtype == COW_BF16) reinterpret_cast<__nv_bfloat16*>(P.out)[at_out] = __float2bfloat16_rn(y);
        else reinterpret_cast<__half*>(P.out)[at_out] = __float2half_rn(y);
      } else {
        partial[h * kRow + d] = v;
        if (d == 0) {
          partial[h * kRow + D] = m;
          partial[h * kRow + D + 1] = l;
        }
      }
    }
    if (!whole) {
      // the block that arrives last joins the pair's parts, in the order of its pages
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        unsigned* word = P.arrived + static_cast<int64_t>(b) * pairs + pair;
        s_last = atomicInc(word, static_cast<unsigned>(sharers - 1)) == static_cast<unsigned>(sharers - 1);
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        for (int i = tid; i < heads_here * D; i += kAttendThreads) {
          const int h = i / D, d = i % D;
          float m = -INFINITY, l = 0.f, v = 0.f;
          for (int k = 0; k < sharers; ++k) {
            const float* r = P.partials + (2 * (first_block + k) + (k == 0 ? 1 : 0)) * (kAttendHeads * kRow) + h * kRow;
            const float rm = __ldcg(r + D), n = fmaxf(m, rm), base = n == -INFINITY ? 0.f : n;
            const float fo = exp2_fast(m - base), fr = exp2_fast(rm - base);
            l = l * fo + __ldcg(r + D + 1) * fr;
            v = v * fo + __ldcg(r + d) * fr;
            m = n;
          }
          const float y = v / l;
          const int64_t at_out = (static_cast<int64_t>(b) * P.heads + head0 + h) * D + d;
          if (P.dtype == COW_F32) reinterpret_cast<float*>(P.out)[at_out] = y;
          else if (P.dtype == COW_BF16) reinterpret_cast<__nv_bfloat16*>(P.out)[at_out] = __float2bfloat16_rn(y);
          else reinterpret_cast<__half*>(P.out)[at_out] = __float2half_rn(y);
        }
      }
    }
    __syncthreads();  // shared memory is free for the next run
  }
}

bool shape_ok(const cow_kv_pages* c) {
  return c->requests >= 0 && c->requests <= COW_MAX_REQUESTS && c->max_blocks >= 0 &&
         c->requests * c->max_blocks < (1 << 25) && c->pages >= 0 && c->pages < (1 << 25) && c->kv_heads >= 1 &&
         c->kv_heads <= 1024 && (c->width == 32 || c->width == 64 || c->width == 96 || c->width == 128);
}
bool rows_ok(const void* p, int64_t s0, int64_t s1, int dtype) {
  const int64_t size = elem_size(dtype);
  return p && aligned16(p) && (s0 * size) % 16 == 0 && (s1 * size) % 16 == 0;
}

template <int DT>
void launch_store(const StoreLaunch& P, int width, dim3 grid, cudaStream_t stream) {
  if (width == 32) cow_kv8_store_kernel<DT, 32><<<grid, kStoreThreads, 0, stream>>>(P);
  else if (width == 64) cow_kv8_store_kernel<DT, 64><<<grid, kStoreThreads, 0, stream>>>(P);
  else if (width == 96) cow_kv8_store_kernel<DT, 96><<<grid, kStoreThreads, 0, stream>>>(P);
  else cow_kv8_store_kernel<DT, 128><<<grid, kStoreThreads, 0, stream>>>(P);
}

using AttendFn = void (*)(const AttendLaunch);

AttendFn attend_fn(int width, bool split) {
  if (width == 32) return split ? cow_kv8_attend_kernel<32, true> : cow_kv8_attend_kernel<32, false>;
  if (width == 64) return split ? cow_kv8_attend_kernel<64, true> : cow_kv8_attend_kernel<64, false>;
  if (width == 96) return split ? cow_kv8_attend_kernel<96, true> : cow_kv8_attend_kernel<96, false>;
  return split ? cow_kv8_attend_kernel<128, true> : cow_kv8_attend_kernel<128, false>;
}

constexpr int kMaxAttendBlocks = 148 * 16;  // partials are sized for this many, more never run

// bytes of the partials, then the arrival words
int64_t partial_bytes(int width) {
  return static_cast<int64_t>(2 * kMaxAttendBlocks) * kAttendHeads * (width + 2) * sizeof(float);
}

}  // namespace

extern "C" {

int cow_kv8_store(const cow_kv_pages* cache, int32_t layer, const void* keys, int64_t key_token_stride,
                  int64_t key_head_stride, const void* values, int64_t value_token_stride, int64_t value_head_stride,
                  int32_t dtype, const int32_t* plan, int64_t tokens, void* stream) {
  if (!cache || !valid_dtype(dtype) || !plan || !aligned16(plan) || layer < 0 || layer >= cache->layers || tokens < 0)
    return COW_ERR_INVALID;
  if (!shape_ok(cache)) return COW_ERR_UNSUPPORTED;
  if (tokens == 0) return COW_OK;
  if (!rows_ok(keys, key_token_stride, key_head_stride, dtype) ||
      !rows_ok(values, value_token_stride, value_head_stride, dtype) || !cache->key_codes || !cache->value_codes ||
      !cache->key_scales || !cache->value_scales)
    return COW_ERR_INVALID;
  const int64_t tiles = layer * cache->pages * cache->kv_heads, size = elem_size(dtype);
  const int64_t bytes = tiles * kPage * cache->width;
  StoreLaunch P{{cache->key_codes + bytes, cache->value_codes + bytes},
                {cache->key_scales + tiles, cache->value_scales + tiles},
                {static_cast<const char*>(keys), static_cast<const char*>(values)},
                {key_token_stride * size, value_token_stride * size},
                {key_head_stride * size, value_head_stride * size},
                plan, cache->kv_heads, static_cast<int32_t>(cache->pages)};
  const int64_t pieces = (tokens < tokens / kPage + 2 * cache->requests) ? tokens : tokens / kPage + 2 * cache->requests;
  const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(cache->kv_heads));
  if (dtype == COW_F32) launch_store<COW_F32>(P, cache->width, grid, as_stream(stream));
  else if (dtype == COW_BF16) launch_store<COW_BF16>(P, cache->width, grid, as_stream(stream));
  else launch_store<COW_F16>(P, cache->width, grid, as_stream(stream));
  return launch_status();
}

int cow_kv8_read(const cow_kv_pages* cache, int32_t layer, const int32_t* slots, int64_t count, void* keys,
                 void* values, int32_t dtype, void* stream) {
  if (!cache || !valid_dtype(dtype) || layer < 0 || layer >= cache->layers || count < 0 || count >= (int64_t{1} << 31))
    return COW_ERR_INVALID;
  if (!shape_ok(cache)) return COW_ERR_UNSUPPORTED;
  if (count == 0) return COW_OK;
  if (!slots || !keys || !values || !aligned16(keys) || !aligned16(values) || !cache->key_codes ||
      !cache->value_codes || !cache->key_scales || !cache->value_scales)
    return COW_ERR_INVALID;
  const int64_t tiles = layer * cache->pages * cache->kv_heads, bytes = tiles * kPage * cache->width;
  ReadLaunch P{{cache->key_codes + bytes, cache->value_codes + bytes},
               {cache->key_scales + tiles, cache->value_scales + tiles},
               {static_cast<char*>(keys), static_cast<char*>(values)},
               slots, count, cache->kv_heads, static_cast<int32_t>(cache->pages), cache->width, dtype};
  const dim3 grid(static_cast<unsigned>((count + kReadSlots - 1) / kReadSlots), static_cast<unsigned>(cache->kv_heads));
  cow_kv8_read_kernel<<<grid, kStoreThreads, 0, as_stream(stream)>>>(P);
  return launch_status();
}

int64_t cow_kv8_attend_workspace_bytes(const cow_kv_pages* cache, int32_t heads) {
  if (!cache || !shape_ok(cache) || heads < 1 || heads % cache->kv_heads) return -1;
  const int64_t chunks = (heads / cache->kv_heads + kAttendHeads - 1) / kAttendHeads;
  return partial_bytes(cache->width) + cache->requests * cache->kv_heads * chunks * static_cast<int64_t>(sizeof(unsigned));
}

int cow_kv8_attend(const cow_kv_pages* cache, int32_t layer, const void* queries, int64_t query_request_stride,
                   int64_t query_head_stride, int32_t dtype, int32_t heads, float scale, void* out, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  if (!cache || !valid_dtype(dtype) || layer < 0 || layer >= cache->layers) return COW_ERR_INVALID;
  if (!shape_ok(cache)) return COW_ERR_UNSUPPORTED;
  const int64_t need = cow_kv8_attend_workspace_bytes(cache, heads);
  if (need < 0 || workspace_bytes < need || !workspace || !aligned16(workspace) || !cache->status) return COW_ERR_INVALID;
  if (cache->requests == 0) return COW_OK;
  if (!rows_ok(queries, query_request_stride, query_head_stride, dtype) || !out || !aligned16(out) || !cache->lengths ||
      (cache->max_blocks > 0 && cache->pages > 0 &&
       (!cache->block_tables || !cache->key_codes || !cache->value_codes || !cache->key_scales || !cache->value_scales)))
    return COW_ERR_INVALID;
  const int64_t max_blocks = cache->pages > 0 ? cache->max_blocks : 0;  // without pages nothing is cached
  const int64_t tiles = layer * cache->pages * cache->kv_heads, bytes = tiles * kPage * cache->width;
  const int group = heads / cache->kv_heads, chunks = (group + kAttendHeads - 1) / kAttendHeads;
  AttendLaunch P{cache->key_codes + bytes, cache->value_codes + bytes, cache->key_scales + tiles,
                 cache->value_scales + tiles, cache->block_tables, cache->lengths, static_cast<const char*>(queries),
                 static_cast<char*>(out), static_cast<float*>(workspace),
                 reinterpret_cast<unsigned*>(static_cast<char*>(workspace) + partial_bytes(cache->width)), cache->status,
                 query_request_stride, query_head_stride, max_blocks, static_cast<int32_t>(cache->requests),
                 cache->kv_heads, heads, group, chunks, static_cast<int32_t>(cache->pages), dtype,
                 scale * 1.4426950408889634f};
  const AttendFn fn = attend_fn(cache->width, dtype == COW_F32);
  // the prefix is sized for whole 1,024s of requests, so that few sizes are ever asked for
  const size_t smem = static_cast<size_t>(kAttendWarps) * 2 * kPage * cache->width +
                      sizeof(int) * ((static_cast<size_t>(cache->requests) / 1024 + 1) * 1024);
  const int resident = resident_blocks(reinterpret_cast<const void*>(fn), kAttendThreads, smem);
  if (!resident) return COW_ERR_CUDA;
  const int64_t most = cache->requests * max_blocks * cache->kv_heads * chunks;
  const int64_t blocks = most < resident ? (most < 1 ? 1 : most) : resident;
  fn<<<static_cast<unsigned>(blocks < kMaxAttendBlocks ? blocks : kMaxAttendBlocks), kAttendThreads, smem,
       as_stream(stream)>>>(P);
  return launch_status();
}

}  // extern "C"
