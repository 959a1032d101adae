// cow_kv8.cu -- the paged K/V cache held in 8 bits: store, read back, attend.
//
// A page holds 64 tokens of one key/value head as e4m3 codes with one scale for its keys and
// one for its values.  Scales are powers of two: a code keeps the same four significant bits
// whatever the scale's mantissa would be, so a finer scale gains nothing, while x / scale
// is exact before its one rounding, and when a later token of the page needs a larger scale,
// the codes already there move to it exactly (but for those that become subnormal).
// Keys lie [token][width]; values lie transposed, [width][token], so that one lane's 16-byte
// word of either is the operand of a matrix instruction without any exchange.  In rows of 128 keys' bytes
// the two halves of odd tokens are exchanged: lanes that read the same half of neighbouring rows
// then meet all banks of shared memory.

#include <cuda_fp8.h>

#include <algorithm>

#include "cow_common.cuh"

namespace {

constexpr int kPage = COW_PAGE_TOKENS;
constexpr int kStoreThreads = 256;
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

// Byte `d` of token t's row in a page's keys.
template <int D>
__device__ __forceinline__ int key_at(int t, int d) {
  return t * D + (D == 128 ? d ^ ((t & 1) << 6) : d);
}

// 16 bytes of a tensor: four 32-bit words of one or two elements
template <int DT>
struct Vec16 {
  static constexpr int kElems = DT == COW_F32 ? 4 : 8;
  static constexpr int kPerWord = kElems / 4;
  static __device__ __forceinline__ void word(unsigned w, float* x) {
    if constexpr (DT == COW_F32) {
      x[0] = __uint_as_float(w);
    } else if constexpr (DT == COW_BF16) {
      x[0] = __uint_as_float(w << 16);
      x[1] = __uint_as_float(w & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
      x[0] = f.x;
      x[1] = f.y;
    }
  }
  static __device__ __forceinline__ void get(uint4 u, float* x) {
    word(u.x, x);
    word(u.y, x + kPerWord);
    word(u.z, x + 2 * kPerWord);
    word(u.w, x + 3 * kPerWord);
  }
};
__device__ __forceinline__ unsigned word_of(uint4 u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

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
// One block per (page piece, head) of the plan and keys or values: the piece's tokens
// are read once into registers, their largest magnitude gives the scale, and the codes are
// written.  Keys: a thread's 16 bytes are neighbours of the next thread's.  Values: a lane
// reads one 16-byte word of each of four neighbouring tokens and so holds whole 32-bit words
// of four codes of the transposed page; two lanes share a 32-byte sector.
// Bound: memory, (element size + 1) bytes for each element of keys and values.  A block's time is mostly
// latency (load, maximum, store), so many must be resident: 66,000 tokens of 8 heads of 128 in bf16 take 81 us with
// 256 threads and five blocks an SM (5.0 TB/s), 100 us with 128 threads and six, 136 us with keys and
// values in one block of 168 registers.

struct StoreLaunch {
  uint8_t* codes[2];  // keys, values: this layer's pages
  float* scales[2];
  const char* x[2];
  int64_t token_stride[2], head_stride[2];  // bytes
  const int32_t* plan;
  int32_t kv_heads, pages;
};

__device__ __forceinline__ float block_most(float most, float* s_most, int lane, int warp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(kFull, most, o));
  if (lane == 0) s_most[warp] = most;
  __syncthreads();
  most = s_most[0];
#pragma unroll
  for (int w = 1; w < kStoreWarps; ++w) most = fmaxf(most, s_most[w]);
  return most;
}

template <int DT, int D>
__global__ void __launch_bounds__(kStoreThreads, DT == COW_F32 ? 3 : 5) cow_kv8_store_kernel(const __grid_constant__ StoreLaunch P) {
  constexpr int E = Vec16<DT>::kElems;
  constexpr int kVecs = D / E;                                          // 16-byte words per token
  constexpr int kKeyVecs = (kPage * kVecs + kStoreThreads - 1) / kStoreThreads;
  constexpr int kGroups = D / (2 * E);                                  // pairs of words per token
  constexpr int kValueGroups = (kGroups + kStoreWarps - 1) / kStoreWarps;
  __shared__ float s_most[kStoreWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y, which = blockIdx.z;
  if (static_cast<int>(blockIdx.x) >= P.plan[0]) return;
  const int4 piece = reinterpret_cast<const int4*>(P.plan + 4)[blockIdx.x];
  const int first = piece.x, tokens = piece.y, page = piece.z, offset = piece.w;
  if (page < 0 || page >= P.pages) return;
  const int64_t tile = static_cast<int64_t>(page) * P.kv_heads + head, stride = P.token_stride[which];
  const char* src = P.x[which] + first * stride + head * P.head_stride[which];
  uint8_t* dst = P.codes[which] + tile * (kPage * D);
  float* scale = P.scales[which] + tile;
  // the scale of a page that holds tokens already
  const int old = offset > 0 ? exponent_of(*scale) : kLeastExponent;

  if (which == 0) {
    uint4 k[kKeyVecs];
#pragma unroll
    for (int i = 0; i < kKeyVecs; ++i) {
      const int n = tid + i * kStoreThreads;
      k[i] = make_uint4(0, 0, 0, 0);
      if (n < tokens * kVecs) k[i] = __ldg(reinterpret_cast<const uint4*>(src + (n / kVecs) * stride) + n % kVecs);
    }
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kKeyVecs; ++i) most = most_of<DT>(k[i], most);
    const int e = max(scale_exponent(block_most(most, s_most, lane, warp)), old);
    if (offset > 0 && e > old) {  // codes that were there move to a larger scale
      const float ratio = e - old > 126 ? 0.f : pow2(old - e);
      for (int i = tid; i < offset * D / 4; i += kStoreThreads) {
        unsigned* word = reinterpret_cast<unsigned*>(dst) + i;
        *word = recode4(*word, ratio);
      }
    }
    const float inv = pow2(-e);
#pragma unroll
    for (int i = 0; i < kKeyVecs; ++i) {
      const int n = tid + i * kStoreThreads;
      if (n < tokens * kVecs) {
        float x[E];
        Vec16<DT>::get(k[i], x);
        unsigned codes[E / 4];
#pragma unroll
        for (int j = 0; j < E; j += 4) codes[j / 4] = encode4(x[j] * inv, x[j + 1] * inv, x[j + 2] * inv, x[j + 3] * inv);
        uint8_t* out = dst + key_at<D>(offset + n / kVecs, n % kVecs * E);
        if constexpr (E == 8) *reinterpret_cast<uint2*>(out) = make_uint2(codes[0], codes[1]);
        else *reinterpret_cast<unsigned*>(out) = codes[0];
      }
    }
    if (tid == 0) *scale = pow2(e);  // past the barrier in block_most: every thread has read the old one
    return;
  }

  const int t0 = (lane >> 1) * 4;  // this lane's four tokens of the page
  uint4 v[kValueGroups][4];
#pragma unroll
  for (int i = 0; i < kValueGroups; ++i) {
    const int g = warp + i * kStoreWarps;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + j - offset;
      v[i][j] = make_uint4(0, 0, 0, 0);
      if (g < kGroups && t >= 0 && t < tokens) v[i][j] = __ldg(reinterpret_cast<const uint4*>(src + t * stride) + 2 * g + (lane & 1));
    }
  }
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < kValueGroups; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) most = most_of<DT>(v[i][j], most);
  const int e = max(scale_exponent(block_most(most, s_most, lane, warp)), old);
  if (offset > 0 && e > old) {
    const float ratio = e - old > 126 ? 0.f : pow2(old - e);
    const int words = (offset + 3) / 4;  // the last may hold bytes of new tokens: those are written after the barrier
    for (int i = tid; i < D * words; i += kStoreThreads) {
      unsigned* word = reinterpret_cast<unsigned*>(dst + (i / words) * kPage) + i % words;
      *word = recode4(*word, ratio);
    }
    __syncthreads();
  }
  const float inv = pow2(-e);
  const int have = min(t0 + 4, offset + tokens) - max(t0, offset);
#pragma unroll
  for (int i = 0; i < kValueGroups; ++i) {
    const int g = warp + i * kStoreWarps;
    if (g < kGroups && have > 0) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float x[4][Vec16<DT>::kPerWord];
#pragma unroll
        for (int j = 0; j < 4; ++j) Vec16<DT>::word(word_of(v[i][j], w), x[j]);
#pragma unroll
        for (int d = 0; d < Vec16<DT>::kPerWord; ++d) {
          const unsigned codes = encode4(x[0][d] * inv, x[1][d] * inv, x[2][d] * inv, x[3][d] * inv);
          uint8_t* out = dst + ((2 * g + (lane & 1)) * E + w * Vec16<DT>::kPerWord + d) * kPage + t0;
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
  }
  if (tid == 0) *scale = pow2(e);
}

// --------------------------------------------------------------------------
// read
// --------------------------------------------------------------------------
//
// One block per (32 list entries, head).  Keys: neighbouring threads take 16-byte words of a row, a row after
// another.  Values: the entries' slots fall into columns, aligned groups of four tokens of a page; a thread
// reads a column's word at four neighbouring widths, turns the 4 x 4 codes about, and they leave
// through shared memory as rows.
// Bound: memory, (1 + element size) bytes for each element.  66,000 tokens of 8 heads of 128 to bf16: 86 us (4.7 TB/s).

struct ReadLaunch {
  const uint8_t* codes[2];
  const float* scales[2];
  char* out[2];
  const int32_t* slots;
  int64_t count;
  int32_t kv_heads, pages;
};

constexpr int kReadSlots = 32;
constexpr int kReadThreads = 128;
static_assert(kReadSlots == 32, "the entries are one warp's");

template <int DT>
__device__ __forceinline__ void store16(char* out, unsigned lo, unsigned hi, float scale) {  // 8 codes; 16 or 32 bytes
  const float2 a = decode2(lo), b = decode2(lo >> 16), c = decode2(hi), d = decode2(hi >> 16);
  const float x[8] = {a.x * scale, a.y * scale, b.x * scale, b.y * scale, c.x * scale, c.y * scale, d.x * scale, d.y * scale};
  if constexpr (DT == COW_F32) {
    reinterpret_cast<float4*>(out)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(out)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == COW_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const unsigned*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const unsigned*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(kReadThreads) cow_kv8_read_kernel(const __grid_constant__ ReadLaunch P) {
  constexpr int kSize = DT == COW_F32 ? 4 : 2;
  constexpr int kVecs = D / 8;        // 8 codes
  constexpr int kRow = D / 4 + 1;     // words of a row of codes in shared memory, off the bank period
  __shared__ unsigned s_codes[kReadSlots * kRow];
  __shared__ int s_slots[kReadSlots];
  __shared__ int4 s_columns[kReadSlots];  // first slot of the four, entry of it, first and number of the tokens asked for
  __shared__ int s_count;
  const int tid = threadIdx.x, head = blockIdx.y;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kReadSlots;
  const int here = static_cast<int>(min(static_cast<int64_t>(kReadSlots), P.count - base));
  if (tid < kReadSlots) {
    int slot = -1;
    if (tid < here) {
      slot = P.slots[base + tid];
      if (slot >= P.pages * kPage) slot = -1;
    }
    s_slots[tid] = slot;
  }
  auto tile_of = [&](int slot) { return static_cast<int64_t>(slot / kPage) * P.kv_heads + head; };
  // values: columns, then their words
  if (tid < kReadSlots) {
    const int slot = s_slots[tid], prev = __shfl_up_sync(kFull, slot, 1);
    const bool leads = slot >= 0 && (tid == 0 || slot != prev + 1 || slot % 4 == 0);
    const unsigned lead = __ballot_sync(kFull, leads), follow = __ballot_sync(kFull, slot >= 0 && !leads);
    if (leads) {
      const int first = slot % 4;
      s_columns[__popc(lead & ((1u << tid) - 1))] =
          make_int4(slot - first, tid - first, first, __ffs(~(tid < 31 ? follow >> (tid + 1) : 0)));
    }
    if (tid == 0) s_count = __popc(lead);
  }
  __syncthreads();
  const int columns = s_count;
#pragma unroll 4
  for (int i = tid; i < columns * (D / 4); i += kReadThreads) {
    const int q = i / columns;
    const int4 col = s_columns[i - q * columns];
    const uint8_t* src = P.codes[1] + tile_of(col.x) * (kPage * D) + 4 * q * kPage + col.x % kPage;
    unsigned w[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) w[d] = __ldg(reinterpret_cast<const unsigned*>(src + d * kPage));
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const unsigned lo = __byte_perm(w[0], w[1], t | (4 + t) << 4), hi = __byte_perm(w[2], w[3], t | (4 + t) << 4);
      if (t >= col.z && t < col.z + col.w) s_codes[(col.y + t) * kRow + q] = __byte_perm(lo, hi, 0x5410);
    }
  }
  // keys, from their rows
  for (int i = tid; i < here * kVecs; i += kReadThreads) {
    const int e = i / kVecs, v = i % kVecs, slot = s_slots[e];
    uint2 w = make_uint2(0, 0);
    float scale = 0.f;
    if (slot >= 0) {
      const int64_t tile = tile_of(slot);
      w = __ldg(reinterpret_cast<const uint2*>(P.codes[0] + tile * (kPage * D) + key_at<D>(slot % kPage, 8 * v)));
      scale = P.scales[0][tile];
    }
    store16<DT>(P.out[0] + ((base + e) * P.kv_heads + head) * (D * kSize) + v * 8 * kSize, w.x, w.y, scale);
  }
  __syncthreads();
  for (int i = tid; i < here * kVecs; i += kReadThreads) {
    const int e = i / kVecs, v = i % kVecs, slot = s_slots[e];
    const bool there = slot >= 0;
    store16<DT>(P.out[1] + ((base + e) * P.kv_heads + head) * (D * kSize) + v * 8 * kSize, there ? s_codes[e * kRow + 2 * v] : 0,
                there ? s_codes[e * kRow + 2 * v + 1] : 0, there ? P.scales[1][tile_of(slot)] : 0.f);
  }
}

// --------------------------------------------------------------------------
// attend
// --------------------------------------------------------------------------
//
// One query token per request, s_j = scale * ks * (q . k_j), o = sum_j softmax(s)_j vs v_j with
// the code's k_j, v_j and the page's ks, vs.  Bound: memory, 2 * width bytes for each cached token
// and key head, everything else is small.  So:
// * the pages of all (request, head) pairs form one list, cut into units whatever the requests' lengths:
//   a large one for each resident warp, then small ones taken as warps get free (SMs reach between 80 % and
//   125 % of the mean rate here, so equal shares alone would wait for the slowest).  A pair inside one unit
//   is answered from registers; parts of a pair go to global memory and a second kernel joins them, in the
//   order of their pages.  (Joined by whichever warp came last instead, each join waited behind the
//   queues of page loads for 10 us, a sixth of the whole time.)
// * where no request has more than kAlignedPages and there are blocks for all pairs, each pair gets a block
//   of its own instead and its warps' parts meet in shared memory;
// * a page's K and its V come by one bulk copy each into the warp's own shared memory, the next page's keys
//   while this page's values are used, on into the next pair; no warp waits for another;
// * e4m3 is exact in f16, so both products run on m16n8k16 with f16 operands and f32 sums: pages are
//   the 16-row operand (tokens, then width), the group's query heads the 8 columns, eight heads
//   to a block.  The tcgen05 form would need the codes widened in shared memory first; here they
//   go from the 16-byte words to operands in registers, and at 4 heads to a key the whole
//   contraction is 1/10 of what this instruction sustains at the memory's rate.
//   Queries are scaled per head by a power of two into f16's range; f32 ones are
//   held as two f16 parts (22 bits), and so are their probabilities.
//   (Widths of a query 2^28 below its largest keep fewer bits: f16's last place lies 2^38 below.)
// * running maximum, sum and output of the softmax stay in f32 registers.  A page's weights are taken relative to its
//   own largest score, so that f16 holds them whatever the others' are; the page's sums join the running ones in f32, where
//   the difference of the maxima and the value scale are one factor.
// Measured (32/8 heads of 128, bf16): 64 requests of 64 to 4,096 tokens 65 us (4.3 TB/s: 54 us of it the first kernel),
// 4 of 65,536 102-104 us (5.2 TB/s, the first kernel 5.9); 16 of 256 to 512 tokens, 4 heads of 32, f32: 9 us, where
// latency is all: 1.7 us until the lengths are scanned, 3.5 us for two pages, 1 us for the warps to meet.

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = 32 * kAttendWarps;
constexpr int kAttendHeads = 8;   // query heads of one block: the matrix instruction's columns
constexpr int kJoin = 8;            // parts a warp of the second kernel reads at once
// Threads of a block of the second kernel: few pairs have many parts each, and many pairs are best all at once.  Both kernels,
// 512,000 tokens of 8 heads of 128, with 512 / 128 threads: 32 pairs 180 / 196 us, 64 186 / 192, 128 187 / 183, 144 185 / 179,
// 256 189 / 175, 512 206 / 182.
constexpr int kJoinFewPairs = 96, kJoinThreadsFew = 512, kJoinThreadsMany = 128;
constexpr int kJoinColumns = 148 * 4;
constexpr int kAlignedPages = 16;  // four pages a warp: less than a join through global memory takes
constexpr float kProbShift = 8.f;  // probabilities are held times 2^8: more of f16's range below the largest
// The output is held over 2^40: sums of the largest values do not overflow before their division, and the least
// scale, 2^-64, leaves the smallest codes' products far above f32's last bit.
constexpr float kOutUnit = 1099511627776.f, kOutUnitLog2 = 40.f;

struct AttendLaunch {
  const uint8_t* key_codes;
  const uint8_t* value_codes;
  const float* key_scales;
  const float* value_scales;
  const int32_t* tables;
  const int32_t* lengths;
  const char* q;
  char* out;
  float* parts;       // [2 * units][rows of the group's heads (width, padded by 4): output, then maximum and sum]
  unsigned* taken;    // [2] units taken, warps done: zero between calls
  int32_t* status;
  int64_t q_request_stride, q_head_stride;  // elements
  int64_t max_blocks;
  int64_t slots;  // 2 * units that fit
  int32_t warps;  // of the first kernel
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
  static constexpr int kBytes = kPage * D;
};

// Pages of request b; the pages before each request (prefix [requests + 1] in shared memory), all of them
// and the most of one request, by a block of kThreads.
__device__ __forceinline__ int pages_of(const AttendLaunch& P, int b) {
  return (min(max(P.lengths[b], 0), static_cast<int>(P.max_blocks) * kPage) + kPage - 1) / kPage;
}
template <int kThreads>
__device__ __forceinline__ int2 scan_pages(const AttendLaunch& P, int* prefix, int2* s_scan) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = P.requests, per = (R + kThreads - 1) / kThreads;
  int sum = 0, longest = 0;
  for (int b = tid * per; b < min(R, (tid + 1) * per); ++b) {
    const int n = pages_of(P, b);
    sum += n;
    longest = max(longest, n);
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(kFull, inc, o);
    if (lane >= o) inc += x;
  }
  longest = __reduce_max_sync(kFull, longest);
  if (lane == 31) s_scan[warp] = make_int2(inc, longest);
  __syncthreads();
  int at = inc - sum, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) at += s_scan[w].x;
    all += s_scan[w].x;
    longest = max(longest, s_scan[w].y);
  }
  for (int b = tid * per; b < min(R, (tid + 1) * per); ++b) {
    prefix[b] = at;
    at += pages_of(P, b);
  }
  if (tid == 0) prefix[R] = all;
  __syncthreads();
  return make_int2(all, longest);
}

// A place in the list of pages: pair `pair` of request `b`, page p of np.
struct Place {
  int b, pair, p, np;
};

__device__ __forceinline__ Place place_of(const int* prefix, int requests, int pairs, int x) {
  int lo = 0, hi = requests;  // the last request that begins at or before x: not an empty one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] * pairs <= x) lo = mid; else hi = mid;
  }
  const int np = prefix[lo + 1] - prefix[lo];
  const int at = x - prefix[lo] * pairs;
  return Place{lo, at / np, at % np, np};
}
__device__ __forceinline__ void store_out(const AttendLaunch& P, int64_t at, float y) {
  if (P.dtype == COW_F32) reinterpret_cast<float*>(P.out)[at] = y;
  else if (P.dtype == COW_BF16) reinterpret_cast<__nv_bfloat16*>(P.out)[at] = __float2bfloat16_rn(y);
  else reinterpret_cast<__half*>(P.out)[at] = __float2half_rn(y);
}

// The list cut into units: `warps` of `first` pages, then of `rest` pages.
struct Units {
  int total, first, rest, warps;
  __device__ __forceinline__ int begin(int u) const {
    return static_cast<int>(min(u < warps ? static_cast<int64_t>(u) * first : static_cast<int64_t>(warps) * first + static_cast<int64_t>(u - warps) * rest,
                                static_cast<int64_t>(total)));
  }
  // The first units get 3/4 of the pages, the others eighths of a warp's share; not more units than the
  // workspace holds parts for.
  static __device__ __forceinline__ Units make(int total, int warps, int64_t slots) {
    const int share = total / warps, first = max(share / 4 * 3 + share % 4 * 3 / 4, 1);
    int rest = max((share + 8) / 8, 2);
    const int room = static_cast<int>(slots / 2) - warps - 1, left = max(total - first * warps, 0);
    if (left > static_cast<int64_t>(rest) * room) rest = left / room + 1;
    return Units{total, first, rest, warps};
  }
  __device__ __forceinline__ int of(int x) const { return x < warps * first ? x / first : warps + (x - warps * first) / rest; }
};

// v + 2^x a, x a part's maximum less the largest: in two halves, as the weight may be below what f32 holds and the
// part's output that far above the others'
__device__ __forceinline__ float4 add_part(float x, float4 a, float4 v) {
  const float half = exp2_fast(0.5f * x);
  return f4_axpy(half, f4_scale(half, a), v);
}

template <int D, int kThreads>
__device__ __forceinline__ void join_parts(const AttendLaunch& P, float (*s_ml)[2], float4 (*s_v)[D / 4], int u0, int sharers, int rows, int h,
                                           int64_t out_row) {
  constexpr int kWarps = kThreads / 32, kWords = D / 4;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t size = rows * (D + 4);
  auto part = [&](int k) { return P.parts + (2 * static_cast<int64_t>(u0 + k) + (k == 0 ? 1 : 0)) * size; };
  float m = -INFINITY, l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = warp; k0 < sharers; k0 += kJoin * kWarps) {
    float4 a[kJoin];  // all loads under way before the first is used
    float2 ml[kJoin];
#pragma unroll
    for (int j = 0; j < kJoin; ++j) {
      ml[j] = make_float2(-INFINITY, 0.f);
      a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + j * kWarps < sharers) {
        const float* r = part(k0 + j * kWarps);
        ml[j] = __ldcg(reinterpret_cast<const float2*>(r + rows * D) + h);
        if (lane < kWords) a[j] = __ldcg(reinterpret_cast<const float4*>(r + h * D) + lane);
      }
    }
    float n = m;
#pragma unroll
    for (int j = 0; j < kJoin; ++j) n = fmaxf(n, ml[j].x);
    const float base = n == -INFINITY ? 0.f : n;
    l *= exp2_fast(m - base);
    v = add_part(m - base, v, make_float4(0.f, 0.f, 0.f, 0.f));
    m = n;
#pragma unroll
    for (int j = 0; j < kJoin; ++j) {
      l = fmaf(exp2_fast(ml[j].x - base), ml[j].y, l);
      v = add_part(ml[j].x - base, a[j], v);
    }
  }
  if (lane < kWords) s_v[warp][lane] = v;
  if (lane == 0) {
    s_ml[warp][0] = m;
    s_ml[warp][1] = l;
  }
  __syncthreads();
  if (tid < kWords) {
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ml[w][0]);
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      l = fmaf(exp2_fast(s_ml[w][0] - base), s_ml[w][1], l);
      v = add_part(s_ml[w][0] - base, s_v[w][tid], v);
    }
    st4_rt(P.out, out_row * D + 4 * tid, f4_scale(kOutUnit / l, v), P.dtype);
  }
  __syncthreads();  // the next pair's parts go there
}

// The same for up to kJoin parts: a thread reads all of them for its words of the pair's output.
template <int D, int kThreads>
__device__ __forceinline__ void join_few(const AttendLaunch& P, int u0, int sharers, int rows, int heads_here, int64_t out_row) {
  const int64_t size = rows * (D + 4);
  for (int t = threadIdx.x; t < heads_here * (D / 4); t += kThreads) {
    const int h = t / (D / 4);
    float4 a[kJoin];
    float2 ml[kJoin];
#pragma unroll
    for (int j = 0; j < kJoin; ++j) {
      ml[j] = make_float2(-INFINITY, 0.f);
      a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j < sharers) {
        const float* r = P.parts + (2 * static_cast<int64_t>(u0 + j) + (j == 0 ? 1 : 0)) * size;
        ml[j] = __ldcg(reinterpret_cast<const float2*>(r + rows * D) + h);
        a[j] = __ldcg(reinterpret_cast<const float4*>(r) + t);
      }
    }
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < kJoin; ++j) m = fmaxf(m, ml[j].x);
    const float base = m == -INFINITY ? 0.f : m;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kJoin; ++j) {
      l = fmaf(exp2_fast(ml[j].x - base), ml[j].y, l);
      v = add_part(ml[j].x - base, a[j], v);
    }
    st4_rt(P.out, out_row * D + 4 * t, f4_scale(kOutUnit / l, v), P.dtype);
  }
}

// Joins the parts of the pairs that lie in several units: a block for a pair of few parts, and one for each
// head of a pair of many.  What depends on the lengths alone is done before the first kernel ends.
template <int D, int kThreads>
__global__ void __launch_bounds__(kThreads) cow_kv8_join_kernel(const __grid_constant__ AttendLaunch P) {
  constexpr int kWarps = kThreads / 32, kWords = D / 4;
  extern __shared__ __align__(16) uint8_t smem[];
  int* s_prefix = reinterpret_cast<int*>(smem);
  __shared__ int2 s_scan[kWarps];
  __shared__ float s_ml[kWarps][2];
  __shared__ float4 s_v[kWarps][kWords];
  const int h = blockIdx.y, pairs = P.kv_heads * P.chunks, rows = min(P.group, kAttendHeads);
  const int2 found = scan_pages<kThreads>(P, s_prefix, s_scan);
  const Units units = Units::make(found.x * pairs, P.warps, P.slots);
  bool waited = false;
  if (found.y > kAlignedPages || P.requests * pairs * kAttendWarps > P.warps) {  // else each pair had its own block
    for (int i = blockIdx.x; i < P.requests * pairs; i += gridDim.x) {
      const int b = i / pairs, pair = i - b * pairs, np = s_prefix[b + 1] - s_prefix[b];
      if (np == 0) continue;
      const int pair0 = s_prefix[b] * pairs + pair * np;
      const int u0 = units.of(pair0), sharers = units.of(pair0 + np - 1) - u0 + 1;
      const int kv_head = P.chunks == 1 ? pair : pair / P.chunks, head0 = (pair - kv_head * P.chunks) * kAttendHeads;
      const int heads_here = min(kAttendHeads, P.group - head0);
      const int64_t row = static_cast<int64_t>(b) * P.heads + kv_head * P.group + head0;
      if (sharers == 1 || h >= (sharers <= kJoin ? 1 : heads_here)) continue;
      if (!waited) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are written
        waited = true;
      }
      if (sharers <= kJoin) join_few<D, kThreads>(P, u0, sharers, rows, heads_here, row);
      else join_parts<D, kThreads>(P, s_ml, s_v, u0, sharers, rows, h, row + h);
    }
  }
  if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");  // this kernel ends after the first
}

template <int D, bool kSplit>
__global__ void __launch_bounds__(kAttendThreads, D > 64 ? 3 : 4) cow_kv8_attend_kernel(const __grid_constant__ AttendLaunch P) {
  using S = PageShape<D>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  uint8_t* s_keys = smem + warp * 2 * S::kBytes;
  uint8_t* s_values = s_keys + S::kBytes;
  int* s_prefix = reinterpret_cast<int*>(smem + kAttendWarps * 2 * S::kBytes);  // [requests + 1] pages before
  __shared__ int2 s_scan[kAttendWarps];
  __shared__ uint64_t s_bars[kAttendWarps][2];  // the warp's keys, values are there
  const int R = P.requests, pairs = P.kv_heads * P.chunks, rows = min(P.group, kAttendHeads);

  if (lane == 0) {
    mbar_init(&s_bars[warp][0], 1);
    mbar_init(&s_bars[warp][1], 1);
  }
  const int most = static_cast<int>(P.max_blocks) * kPage;
  const int2 found = scan_pages<kAttendThreads>(P, s_prefix, s_scan);
  const int all = found.x, longest = found.y;

  // a request without tokens: zeros
  for (int b = blockIdx.x; b < R; b += gridDim.x) {
    if (s_prefix[b + 1] == s_prefix[b])
      for (int i = tid; i < P.heads * D / 4; i += kAttendThreads)
        st4_rt(P.out, static_cast<int64_t>(b) * P.heads * D + 4 * i, make_float4(0.f, 0.f, 0.f, 0.f), P.dtype);
  }

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // this warp's first unit of the list
  const int total = all * pairs, warps = gridDim.x * kAttendWarps;
  const bool aligned = longest <= kAlignedPages && R * pairs <= static_cast<int>(gridDim.x);
  const Units units = Units::make(total, warps, P.slots);
  int unit = blockIdx.x * kAttendWarps + warp, x0 = 0, x1 = 0;
  if (aligned) {
    const int b = blockIdx.x / pairs;
    if (b < R) {
      const int np = s_prefix[b + 1] - s_prefix[b];
      x0 = s_prefix[b] * pairs + blockIdx.x % pairs * np;
      x1 = x0 + np * (warp + 1) / kAttendWarps;
      x0 += np * warp / kAttendWarps;
    }
  } else {
    x0 = units.begin(unit);
    x1 = units.begin(unit + 1);
  }

  // Lane i holds entry held_from + i of the block table of the pair that was last asked for.
  int held = 0, held_from = 0;
  auto tile_of = [&](const Place& w, bool new_pair) {
    if (new_pair || w.p - held_from >= 32) {
      held_from = w.p;
      if (held_from + lane < w.np) held = P.tables[w.b * P.max_blocks + held_from + lane];
    }
    int page = __shfl_sync(kFull, held, w.p - held_from);
    if (page < 0 || page >= P.pages) {
      if (lane == 0) atomicOr(P.status, COW_ST_ROW_RANGE);
      page = 0;
    }
    return static_cast<int64_t>(page) * P.kv_heads + w.pair / P.chunks;
  };
  uint64_t* bars = s_bars[warp];
  auto copy = [&](int which, int64_t tile) {  // what was in its place has been read by all lanes
    __syncwarp();
    if (lane == 0) {
      mbar_arrive_expect_tx(&bars[which], S::kBytes);
      bulk_row_copy(which ? s_values : s_keys, (which ? P.value_codes : P.key_codes) + tile * S::kBytes, S::kBytes, &bars[which]);
    }
  };

  if (x0 < x1) {
    Place now = place_of(s_prefix, R, pairs, x0);
    const int64_t tile = tile_of(now, true);
    copy(0, tile);
    copy(1, tile);
    unsigned parity = 0;
    float ks = P.key_scales[tile], vs = P.value_scales[tile];
    unsigned grabbed = 0;  // lane 0: the unit after this one
    if (!aligned && lane == 0) grabbed = atomicAdd(P.taken, 1u);
    bool began = now.p == 0;  // the pair's first page is in this unit

    unsigned qa[S::kKeySteps][2], qb[kSplit ? S::kKeySteps : 1][2];
    float f0 = 0.f, f1 = 0.f, m0 = 0.f, m1 = 0.f, l0 = 0.f, l1 = 0.f;
    float o[D / 16][4];
    int length = 0;
    bool fresh = true;
    // A wait that gave up is reported; what is on its way gets as long again, no copy follows it, and the warp's
    // outputs from there on are NaN.
    bool lost = false;
    auto wait = [&](int which, unsigned phase, bool next_keys) {
      if (lost || __all_sync(kFull, mbar_wait(&bars[which], phase, kSpinLimit))) return;
      lost = true;
      if (lane == 0) atomicOr(P.status, COW_ST_WAIT_TIMEOUT);
      if (!which || next_keys) mbar_wait(&bars[0], which ? phase ^ 1 : phase, kSpinLimit);
      mbar_wait(&bars[1], phase, kSpinLimit);
    };

    for (int x = x0;;) {
      if (fresh) {
        // a new pair: the query of column g as operand columns, scaled so that its largest element is in [2^14, 2^15)
        length = min(P.lengths[now.b], most);
        const int head0 = now.pair / P.chunks * P.group + now.pair % P.chunks * kAttendHeads;
        const bool there = g < min(kAttendHeads, P.group - now.pair % P.chunks * kAttendHeads);
        const int64_t row = now.b * P.q_request_stride + static_cast<int64_t>(head0 + (there ? g : 0)) * P.q_head_stride;
        float v[S::kKeySteps][4];
        float big = 0.f;
#pragma unroll
        for (int k = 0; k < S::kKeySteps; ++k) {
          const int h = k / 4;
          const int d = h < S::kWhole ? 64 * h + 16 * c + 4 * (k % 4) : 64 * S::kWhole + 8 * c + 4 * (k % 2);
          const float4 q = ld4_rt(P.q, row + d, P.dtype);
          v[k][0] = there ? q.x : 0.f;
          v[k][1] = there ? q.y : 0.f;
          v[k][2] = there ? q.z : 0.f;
          v[k][3] = there ? q.w : 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (fabsf(v[k][i]) < INFINITY) big = fmaxf(big, fabsf(v[k][i]));
        }
        big = fmaxf(big, __shfl_xor_sync(kFull, big, 1));
        big = fmaxf(big, __shfl_xor_sync(kFull, big, 2));
        const int e = min(14 - exponent_of(big), 100);
        const float up = pow2(e), unscale = pow2(-e) * P.scale_log2;
#pragma unroll
        for (int k = 0; k < S::kKeySteps; ++k) {
          qa[k][0] = pack_half2(v[k][0] * up, v[k][1] * up);
          qa[k][1] = pack_half2(v[k][2] * up, v[k][3] * up);
          if constexpr (kSplit) {
            qb[k][0] = pack_rest2(v[k][0] * up, v[k][1] * up, qa[k][0]);
            qb[k][1] = pack_rest2(v[k][2] * up, v[k][3] * up, qa[k][1]);
          }
        }
        // this lane's score columns are heads 2c and 2c + 1
        f0 = __shfl_sync(kFull, unscale, 8 * c);
        f1 = __shfl_sync(kFull, unscale, 8 * c + 4);
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        fresh = false;
      }

      // the next page, maybe of the next pair or unit
      const bool unit_ends = x + 1 == x1;
      bool more = !unit_ends;
      Place next = now;
      int64_t next_tile = 0;
      int next_unit = unit, next_x = x + 1;
      if (!unit_ends) {
        if (++next.p == next.np) {
          next.p = 0;
          if (++next.pair == pairs) {
            next.pair = 0;
            do ++next.b;
            while (s_prefix[next.b + 1] == s_prefix[next.b]);  // there is another page, so another request
            next.np = s_prefix[next.b + 1] - s_prefix[next.b];
          }
        }
      } else if (!aligned) {
        next_unit = warps + static_cast<int>(__shfl_sync(kFull, grabbed, 0));
        next_x = units.begin(next_unit);
        more = next_x < total;
        if (more) next = place_of(s_prefix, R, pairs, next_x);
      }
      if (more) {
        const bool new_pair = next.pair != now.pair || next.b != now.b || unit_ends;
        next_tile = tile_of(next, new_pair);
        if (new_pair) {  // its queries, on their way to where the next turn reads them
          const int h = next.pair / P.chunks * P.group + next.pair % P.chunks * kAttendHeads + min(g, min(kAttendHeads, P.group - next.pair % P.chunks * kAttendHeads) - 1);
          const char* q = P.q + (next.b * P.q_request_stride + h * P.q_head_stride) * (P.dtype == COW_F32 ? 4 : 2);
          for (int d = 128 * c; d < D * (P.dtype == COW_F32 ? 4 : 2); d += 512) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + d));
        }
      }

      wait(0, parity, false);
      float s[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
        const int token = (g >> 1) * 16 + 4 * t + (g & 1);
#pragma unroll
        for (int h = 0; h < S::kWhole; ++h) {
          const uint4 a = *reinterpret_cast<const uint4*>(s_keys + key_at<D>(token, 64 * h + 16 * c));
          const uint4 z = *reinterpret_cast<const uint4*>(s_keys + key_at<D>(token + 2, 64 * h + 16 * c));
          const unsigned aw[4] = {a.x, a.y, a.z, a.w}, zw[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const unsigned a0 = lo2(aw[q]), a1 = lo2(zw[q]), a2 = hi2(aw[q]), a3 = hi2(zw[q]);
            mma_f16(s[t], a0, a1, a2, a3, qa[4 * h + q][0], qa[4 * h + q][1]);
            if constexpr (kSplit) mma_f16(s[t], a0, a1, a2, a3, qb[4 * h + q][0], qb[4 * h + q][1]);
          }
        }
        if constexpr (S::kHalf) {
          const uint2 a = *reinterpret_cast<const uint2*>(s_keys + key_at<D>(token, 64 * S::kWhole + 8 * c));
          const uint2 z = *reinterpret_cast<const uint2*>(s_keys + key_at<D>(token + 2, 64 * S::kWhole + 8 * c));
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
      if (more && !lost) copy(0, next_tile);

      // scores, the page's maximum, probabilities
      const int left = length - now.p * kPage;  // tokens of this page, if below 64
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
      for (int y = 4; y < 32; y <<= 1) {
        big0 = fmaxf(big0, __shfl_xor_sync(kFull, big0, y));
        big1 = fmaxf(big1, __shfl_xor_sync(kFull, big1, y));
      }
      const float n0 = fmaxf(m0, big0), n1 = fmaxf(m1, big1);
      // where every score of the page, or so far, is -inf, exponents are taken from 0: probabilities 0, no NaN
      const float b0 = big0 == -INFINITY ? 0.f : big0, b1 = big1 == -INFINITY ? 0.f : big1;
      const float c0 = n0 == -INFINITY ? 0.f : n0, c1 = n1 == -INFINITY ? 0.f : n1;
      const float a0 = exp2_fast(m0 - c0), a1 = exp2_fast(m1 - c1), r0 = exp2_fast(big0 - c0), r1 = exp2_fast(big1 - c1);
      m0 = n0;
      m1 = n1;
      float sum0 = 0.f, sum1 = 0.f;
      unsigned pa[4][2], pb[kSplit ? 4 : 1][2];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float e0 = exp2_fast(s[t][0] - b0 + kProbShift), e1 = exp2_fast(s[t][1] - b1 + kProbShift);
        const float e2 = exp2_fast(s[t][2] - b0 + kProbShift), e3 = exp2_fast(s[t][3] - b1 + kProbShift);
        sum0 += e0 + e2;
        sum1 += e1 + e3;
        const unsigned u0 = pack_half2(e0, e1), u1 = pack_half2(e2, e3);
        pa[t][0] = transpose8x8(u0);
        pa[t][1] = transpose8x8(u1);
        if constexpr (kSplit) {
          pb[t][0] = transpose8x8(pack_rest2(e0, e1, u0));
          pb[t][1] = transpose8x8(pack_rest2(e2, e3, u1));
        }
      }
      l0 = fmaf(l0, a0, sum0 * r0);
      l1 = fmaf(l1, a1, sum1 * r1);
      // one power of two for both: a page's weight may be below what f32 holds and its values that far above the others'
      const float vs_log2 = static_cast<float>(exponent_of(vs)) - kOutUnitLog2;
      const float y0 = exp2_fast(big0 - c0 + vs_log2), y1 = exp2_fast(big1 - c1 + vs_log2);

      wait(1, parity, more);
      parity ^= 1;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint4 a = *reinterpret_cast<const uint4*>(s_values + (16 * i + g) * kPage + 16 * c);
        const uint4 z = *reinterpret_cast<const uint4*>(s_values + (16 * i + 8 + g) * kPage + 16 * c);
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
        // The page's sum apart, then added in f32: the matrix unit's own adds do not round to nearest, and
        // over thousands of pages that would show.
        float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const unsigned v0 = lo2(aw[t]), v1 = lo2(zw[t]), v2 = hi2(aw[t]), v3 = hi2(zw[t]);
          if constexpr (kSplit) mma_f16(y, v0, v1, v2, v3, pb[t][0], pb[t][1]);
          mma_f16(y, v0, v1, v2, v3, pa[t][0], pa[t][1]);
        }
        o[i][0] = fmaf(o[i][0], a0, y[0] * y0);
        o[i][1] = fmaf(o[i][1], a1, y[1] * y1);
        o[i][2] = fmaf(o[i][2], a0, y[2] * y0);
        o[i][3] = fmaf(o[i][3], a1, y[3] * y1);
      }
      if (more) {
        if (!lost) copy(1, next_tile);
        ks = P.key_scales[next_tile];
        vs = P.value_scales[next_tile];
      }

      const bool ended = now.p + 1 == now.np;
      if (ended || unit_ends) {
        // the pair, or this unit's part of it, is done
#pragma unroll
        for (int y = 4; y < 32; y <<= 1) {
          l0 += __shfl_xor_sync(kFull, l0, y);
          l1 += __shfl_xor_sync(kFull, l1, y);
        }
        if (lost) l0 = l1 = __int_as_float(0x7fc00000);
        const int chunk = now.pair % P.chunks, heads_here = min(kAttendHeads, P.group - chunk * kAttendHeads);
        const int64_t row = static_cast<int64_t>(now.b) * P.heads + now.pair / P.chunks * P.group + chunk * kAttendHeads;
        if (began && ended && !aligned) {
          const float y0 = kOutUnit / l0, y1 = kOutUnit / l1;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            if (2 * c < heads_here) {
              store_out(P, (row + 2 * c) * D + 16 * i + g, o[i][0] * y0);
              store_out(P, (row + 2 * c) * D + 16 * i + g + 8, o[i][2] * y0);
            }
            if (2 * c + 1 < heads_here) {
              store_out(P, (row + 2 * c + 1) * D + 16 * i + g, o[i][1] * y1);
              store_out(P, (row + 2 * c + 1) * D + 16 * i + g + 8, o[i][3] * y1);
            }
          }
        } else {
          if (aligned) __syncwarp();  // this warp's pages are used up
          float* mine = aligned ? reinterpret_cast<float*>(s_keys) : P.parts + static_cast<int64_t>(2 * unit + (began ? 1 : 0)) * (rows * (D + 4));
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            if (2 * c < rows) {
              mine[(2 * c) * D + 16 * i + g] = o[i][0];
              mine[(2 * c) * D + 16 * i + g + 8] = o[i][2];
            }
            if (2 * c + 1 < rows) {
              mine[(2 * c + 1) * D + 16 * i + g] = o[i][1];
              mine[(2 * c + 1) * D + 16 * i + g + 8] = o[i][3];
            }
          }
          if (g == 0) {
            float2* ml = reinterpret_cast<float2*>(mine + rows * D);
            if (2 * c < rows) ml[2 * c] = make_float2(m0, l0);
            if (2 * c + 1 < rows) ml[2 * c + 1] = make_float2(m1, l1);
          }
        }
        began = true;
        fresh = true;
      }
      if (!more) break;
      if (unit_ends) {
        unit = next_unit;
        x1 = units.begin(unit + 1);
        began = next.p == 0;
        if (lane == 0) grabbed = atomicAdd(P.taken, 1u);
      }
      x = next_x;
      now = next;
    }
  }

  if (!aligned) {
    // the last warp to end leaves the count of units as it was
    if (lane == 0) {
      __threadfence();
      if (atomicInc(P.taken + 1, static_cast<unsigned>(warps - 1)) == static_cast<unsigned>(warps - 1)) *P.taken = 0;
    }
    return;
  }
  // ---- the warps' parts of the block's pair
  const int b = blockIdx.x / pairs, pair = blockIdx.x % pairs;
  if (b >= R || s_prefix[b + 1] == s_prefix[b]) return;  // the whole block
  __syncthreads();
  const int np = s_prefix[b + 1] - s_prefix[b];
  const int chunk = pair % P.chunks, heads_here = min(kAttendHeads, P.group - chunk * kAttendHeads);
  const int64_t row = static_cast<int64_t>(b) * P.heads + pair / P.chunks * P.group + chunk * kAttendHeads;
  for (int t = tid; t < heads_here * (D / 4); t += kAttendThreads) {
    const int h = t / (D / 4);
    float m = -INFINITY, l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kAttendWarps; ++w) {
      if (np * w / kAttendWarps == np * (w + 1) / kAttendWarps) continue;  // no page
      const float* part = reinterpret_cast<const float*>(smem + w * 2 * S::kBytes);
      const float2 ml = reinterpret_cast<const float2*>(part + rows * D)[h];
      const float n = fmaxf(m, ml.x), base = n == -INFINITY ? 0.f : n;
      l = l * exp2_fast(m - base) + ml.y * exp2_fast(ml.x - base);
      v = add_part(m - base, v, add_part(ml.x - base, reinterpret_cast<const float4*>(part)[t], make_float4(0.f, 0.f, 0.f, 0.f)));
      m = n;
    }
    st4_rt(P.out, row * D + 4 * t, f4_scale(kOutUnit / l, v), P.dtype);
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

template <int DT>
void launch_read(const ReadLaunch& P, int width, dim3 grid, cudaStream_t stream) {
  if (width == 32) cow_kv8_read_kernel<DT, 32><<<grid, kReadThreads, 0, stream>>>(P);
  else if (width == 64) cow_kv8_read_kernel<DT, 64><<<grid, kReadThreads, 0, stream>>>(P);
  else if (width == 96) cow_kv8_read_kernel<DT, 96><<<grid, kReadThreads, 0, stream>>>(P);
  else cow_kv8_read_kernel<DT, 128><<<grid, kReadThreads, 0, stream>>>(P);
}

using AttendFn = void (*)(const AttendLaunch);

AttendFn attend_fn(int width, bool split) {
  if (width == 32) return split ? cow_kv8_attend_kernel<32, true> : cow_kv8_attend_kernel<32, false>;
  if (width == 64) return split ? cow_kv8_attend_kernel<64, true> : cow_kv8_attend_kernel<64, false>;
  if (width == 96) return split ? cow_kv8_attend_kernel<96, true> : cow_kv8_attend_kernel<96, false>;
  return split ? cow_kv8_attend_kernel<128, true> : cow_kv8_attend_kernel<128, false>;
}

template <int kThreads>
AttendFn join_fn(int width) {
  if (width == 32) return cow_kv8_join_kernel<32, kThreads>;
  if (width == 64) return cow_kv8_join_kernel<64, kThreads>;
  return width == 96 ? cow_kv8_join_kernel<96, kThreads> : cow_kv8_join_kernel<128, kThreads>;
}

// Blocks of a launch at most: what 168 (128) registers a thread let an SM hold.
int max_attend_blocks(int width) { return 148 * (width > 64 ? 3 : 4); }
// Units of W warps: W of floor(3/4 of a warp's share), at least 1, and what is left in eighths of a share
// rounded up, at least 2.  Left are at most total / 4 + W pages: with total <= 16 W 2.5 W units of 2, above it
// (total / 4 + W) / (total / 8 W) <= 2.5 W, and one that is not full.
int64_t max_units(int width) { return int64_t{4} * max_attend_blocks(width) * kAttendWarps; }
int64_t parts_bytes(int width, int group) {
  return 2 * max_units(width) * (group < kAttendHeads ? group : kAttendHeads) * (width + 4) * static_cast<int64_t>(sizeof(float));
}

}  // namespace

extern "C" {

int cow_kv8_store(const cow_kv_pages* cache, int32_t layer, const void* keys, int64_t key_token_stride,
                  int64_t key_head_stride, const void* values, int64_t value_token_stride, int64_t value_head_stride,
                  int32_t dtype, const int32_t* plan, int64_t tokens, void* stream) {
  if (!cache || !valid_dtype(dtype) || !plan || !aligned16(plan) || layer < 0 || layer >= cache->layers || tokens < 0)
    return COW_ERR_INVALID;
  if (!shape_ok(cache)) return COW_ERR_UNSUPPORTED;
  const int64_t pieces = std::min(tokens, tokens / kPage + 2 * cache->requests);  // at most; none without requests
  if (pieces == 0) return COW_OK;
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
  const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(cache->kv_heads), 2);
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
               slots, count, cache->kv_heads, static_cast<int32_t>(cache->pages)};
  const dim3 grid(static_cast<unsigned>((count + kReadSlots - 1) / kReadSlots), static_cast<unsigned>(cache->kv_heads));
  if (dtype == COW_F32) launch_read<COW_F32>(P, cache->width, grid, as_stream(stream));
  else if (dtype == COW_BF16) launch_read<COW_BF16>(P, cache->width, grid, as_stream(stream));
  else launch_read<COW_F16>(P, cache->width, grid, as_stream(stream));
  return launch_status();
}

int64_t cow_kv8_attend_workspace_bytes(const cow_kv_pages* cache, int32_t heads) {
  if (!cache || !shape_ok(cache) || heads < 1 || heads % cache->kv_heads) return -1;
  return 16 + parts_bytes(cache->width, heads / cache->kv_heads);
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
       (!cache->block_tables || !cache->key_codes || !cache->value_codes || !aligned16(cache->key_codes) ||
        !aligned16(cache->value_codes) || !cache->key_scales || !cache->value_scales)))
    return COW_ERR_INVALID;
  const int64_t max_blocks = cache->pages > 0 ? cache->max_blocks : 0;  // without pages nothing is cached
  const int64_t tiles = layer * cache->pages * cache->kv_heads, bytes = tiles * kPage * cache->width;
  const int group = heads / cache->kv_heads, chunks = (group + kAttendHeads - 1) / kAttendHeads;
  const AttendFn fn = attend_fn(cache->width, dtype == COW_F32);
  // the prefix is sized for whole 512s of requests, so that few sizes are ever asked for
  const size_t smem = static_cast<size_t>(kAttendWarps) * 2 * kPage * cache->width +
                      sizeof(int) * ((static_cast<size_t>(cache->requests) / 512 + 1) * 512);
  const int resident = resident_blocks(reinterpret_cast<const void*>(fn), kAttendThreads, smem);
  if (!resident) return COW_ERR_CUDA;
  const int64_t most = cache->requests * max_blocks * cache->kv_heads * chunks;
  if (most >= (int64_t{1} << 31) - (1 << 20) || cache->requests * cache->kv_heads * chunks >= (1 << 28)) return COW_ERR_UNSUPPORTED;
  int64_t blocks = most < 1 ? 1 : most;
  if (blocks > resident) blocks = resident;
  if (blocks > max_attend_blocks(cache->width)) blocks = max_attend_blocks(cache->width);
  const AttendLaunch P{cache->key_codes + bytes, cache->value_codes + bytes, cache->key_scales + tiles,
                       cache->value_scales + tiles, cache->block_tables, cache->lengths, static_cast<const char*>(queries),
                       static_cast<char*>(out), reinterpret_cast<float*>(static_cast<char*>(workspace) + 16),
                       static_cast<unsigned*>(workspace), cache->status, query_request_stride, query_head_stride, max_blocks,
                       2 * max_units(cache->width), static_cast<int32_t>(blocks * kAttendWarps),
                       static_cast<int32_t>(cache->requests), cache->kv_heads, heads, group, chunks,
                       static_cast<int32_t>(cache->pages), dtype, scale * 1.4426950408889634f};
  fn<<<static_cast<unsigned>(blocks), kAttendThreads, smem, as_stream(stream)>>>(P);
  if (launch_status() != COW_OK) return COW_ERR_CUDA;
  // tables so short that every pair has a block of its own: nothing to join
  if (max_blocks <= kAlignedPages && cache->requests * cache->kv_heads * chunks <= blocks) return COW_OK;
  cudaLaunchConfig_t cfg = {};
  const int rows = group < kAttendHeads ? group : kAttendHeads;
  const int64_t all_pairs = cache->requests * cache->kv_heads * chunks, wide = kJoinColumns;
  cfg.gridDim = dim3(static_cast<unsigned>(all_pairs < wide ? all_pairs : wide), static_cast<unsigned>(rows));
  cfg.dynamicSmemBytes = sizeof(int) * (static_cast<size_t>(cache->requests) + 1);
  const bool few = all_pairs <= kJoinFewPairs;
  cfg.blockDim = dim3(few ? kJoinThreadsFew : kJoinThreadsMany);
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, few ? join_fn<kJoinThreadsFew>(cache->width) : join_fn<kJoinThreadsMany>(cache->width), P);
  return launch_status();
}

}  // extern "C"
