// cow_pages.cu -- block tables and slot maps of the paged K/V cache, from request lengths.
//
// With P(n) = ceil(n / 64), moving request b from cur_b to target_b tokens frees its
// blocks P(target_b) .. P(cur_b)-1 or takes blocks P(cur_b) .. P(target_b)-1.  With
// exclusive prefix sums over the requests of the blocks freed (F in all), the blocks taken
// (T), the new tokens and their page pieces, every output word has a closed form:
//   the k-th page freed goes to   free_pages[count + F - 1 - k]
//   the r-th page taken is        the r-th freed one for r < F, else free_pages[count - 1 - (r - F)]
//   new token t of request b at position p has slot 64 * page(b, p / 64) + p % 64
// so no word depends on another block's output, and one launch does it without a wait:
// every block of threads reads the lengths, targets and tables as they were, scans them for
// itself (8 bytes a request), and writes its share of the outputs.  What the others may still
// read (lengths, the count, the table entries of freed pages that are taken again in the
// same call) is changed by the block that arrives last.
//
// Bound: launch latency and two rounds of dependent loads for a decode step (64 requests: 6 us on the
// device, 10 us a call with the host's part); for admissions the 8 bytes a token of the slot and position maps
// (1,024 requests with 1.06 million new tokens: 15 us, 0.6 TB/s, half of it the scan that every block repeats
// instead of waiting for another's).

#include "cow_common.cuh"

namespace {

constexpr int kResizeThreads = 512;
constexpr int kTokensPerThread = 4;

struct ResizeLaunch {
  int32_t* tables;
  int32_t* lengths;
  int32_t* free_pages;
  int32_t* free_count;
  int32_t* status;
  int32_t* ticket;
  const int32_t* targets;
  int32_t* head;       // [4]
  int4* pieces;        // [max_pieces]
  int32_t* starts;     // [requests + 1]
  int32_t* slots;      // [tokens]
  int32_t* positions;  // [tokens]
  int64_t max_blocks;
  int32_t requests, tokens, max_pieces, pages;
};

__device__ __forceinline__ int page_count(int n) { return (n + COW_PAGE_TOKENS - 1) / COW_PAGE_TOKENS; }

// The last request whose prefix is <= x: with x below the total, the one x belongs to.
__device__ __forceinline__ int owner_of(const int* prefix, int requests, int x) {
  int lo = 0, hi = requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kResizeThreads) cow_pages_resize_kernel(const __grid_constant__ ResizeLaunch P) {
  extern __shared__ int smem[];
  const int R = P.requests, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* s_cur = smem;               // [R]
  int* s_target = s_cur + R;       // [R]
  int* s_new = s_target + R;       // [R + 1] prefixes
  int* s_taken = s_new + R + 1;    // [R + 1]
  int* s_freed = s_taken + R + 1;  // [R + 1]
  int* s_piece = s_freed + R + 1;  // [R + 1]
  __shared__ int4 s_warp[kResizeThreads / 32];
  __shared__ int s_bad, s_last;
  if (tid == 0) s_bad = 0;
  __syncthreads();

  // each thread owns `per` consecutive requests
  const int per = (R + kResizeThreads - 1) / kResizeThreads;
  const int most = static_cast<int>(P.max_blocks) * COW_PAGE_TOKENS;
  const int count = *P.free_count;
  int4 sum = make_int4(0, 0, 0, 0);  // new tokens, taken, freed, pieces
  bool bad = false;
  for (int b = tid * per; b < min(R, (tid + 1) * per); ++b) {
    int cur = P.lengths[b], target = P.targets[b];
    if (cur < 0 || cur > most || target < 0 || target > most) {
      bad = true;
      cur = target = 0;
    }
    s_cur[b] = cur;
    s_target[b] = target;
    const int had = page_count(cur), wants = page_count(target);
    sum.x += max(target - cur, 0);
    sum.y += max(wants - had, 0);
    sum.z += max(had - wants, 0);
    sum.w += target > cur ? wants - cur / COW_PAGE_TOKENS : 0;
  }
  if (bad) s_bad = 1;
  int4 inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(kFull, inc.x, o), y = __shfl_up_sync(kFull, inc.y, o);
    const int z = __shfl_up_sync(kFull, inc.z, o), w = __shfl_up_sync(kFull, inc.w, o);
    if (lane >= o) inc = make_int4(inc.x + x, inc.y + y, inc.z + z, inc.w + w);
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  int4 at = make_int4(inc.x - sum.x, inc.y - sum.y, inc.z - sum.z, inc.w - sum.w), all = make_int4(0, 0, 0, 0);
  for (int w = 0; w < kResizeThreads / 32; ++w) {
    const int4 v = s_warp[w];
    if (w < warp) at = make_int4(at.x + v.x, at.y + v.y, at.z + v.z, at.w + v.w);
    all = make_int4(all.x + v.x, all.y + v.y, all.z + v.z, all.w + v.w);
  }
  for (int b = tid * per; b < min(R, (tid + 1) * per); ++b) {
    const int cur = s_cur[b], target = s_target[b], had = page_count(cur), wants = page_count(target);
    s_new[b] = at.x;
    s_taken[b] = at.y;
    s_freed[b] = at.z;
    s_piece[b] = at.w;
    at.x += max(target - cur, 0);
    at.y += max(wants - had, 0);
    at.z += max(had - wants, 0);
    at.w += target > cur ? wants - cur / COW_PAGE_TOKENS : 0;
  }
  if (tid == 0) {
    s_new[R] = all.x;
    s_taken[R] = all.y;
    s_freed[R] = all.z;
    s_piece[R] = all.w;
  }
  __syncthreads();

  const int freed = all.z, taken = all.y;
  int error = s_bad ? COW_ST_INDEX_RANGE : 0;
  if (all.x > P.tokens || all.w > P.max_pieces) error |= COW_ST_PLAN_TOKENS;
  if (count < 0 || count + static_cast<int64_t>(freed) > P.pages || taken > count + static_cast<int64_t>(freed))
    error |= COW_ST_SLAB_EXHAUSTED;
  const bool mixed = freed > 0 && taken > 0;
  const int threads = gridDim.x * kResizeThreads, self = blockIdx.x * kResizeThreads + tid;

  auto freed_page = [&](int k) {
    const int b = owner_of(s_freed, R, k);
    return P.tables[b * P.max_blocks + page_count(s_target[b]) + (k - s_freed[b])];
  };
  auto taken_page = [&](int r) { return r < freed ? freed_page(r) : P.free_pages[count - 1 - (r - freed)]; };
  auto page_of = [&](int b, int block) {
    const int had = page_count(s_cur[b]);
    return block < had ? P.tables[b * P.max_blocks + block] : taken_page(s_taken[b] + block - had);
  };

  if (error) {
    if (self == 0) {
      atomicOr(P.status, error);
      *reinterpret_cast<int4*>(P.head) = make_int4(0, 0, 0, 0);
    }
    for (int b = self; b <= R; b += threads) P.starts[b] = 0;
    for (int64_t t = self; t < P.tokens; t += threads) P.slots[t] = P.positions[t] = -1;
    return;  // the same decision in every block: nobody takes a ticket
  }

  if (self == 0) *reinterpret_cast<int4*>(P.head) = make_int4(all.w, all.x, 0, 0);
  for (int b = self; b <= R; b += threads) P.starts[b] = s_new[b];
  // new table entries (never read as old ones) and the stack's new top
  for (int r = self; r < taken; r += threads) {
    const int b = owner_of(s_taken, R, r);
    P.tables[b * P.max_blocks + page_count(s_cur[b]) + (r - s_taken[b])] = taken_page(r);
  }
  for (int k = self; k < freed; k += threads) {
    const int b = owner_of(s_freed, R, k);
    int32_t* entry = P.tables + b * P.max_blocks + page_count(s_target[b]) + (k - s_freed[b]);
    P.free_pages[count + freed - 1 - k] = *entry;
    if (!mixed) *entry = -1;
  }
  for (int i = self; i < all.w; i += threads) {
    const int b = owner_of(s_piece, R, i), cur = s_cur[b], target = s_target[b];
    const int block = cur / COW_PAGE_TOKENS + (i - s_piece[b]);
    const int from = max(cur, block * COW_PAGE_TOKENS), to = min(target, (block + 1) * COW_PAGE_TOKENS);
    P.pieces[i] = make_int4(s_new[b] + from - cur, to - from, page_of(b, block), from % COW_PAGE_TOKENS);
  }
  // kTokensPerThread neighbouring tokens share the search and mostly the page.  (In 64 bits: the announced tokens may be near
  // 2^31, where an int would wrap at the last step.)
  for (int64_t first = int64_t{self} * kTokensPerThread; first < P.tokens; first += int64_t{threads} * kTokensPerThread) {
    const int t0 = static_cast<int>(first), end = static_cast<int>(min(first + kTokensPerThread, static_cast<int64_t>(P.tokens)));
    int b = t0 < all.x ? owner_of(s_new, R, t0) : R, block = -1, page = 0;
    for (int t = t0; t < end; ++t) {
      if (t >= all.x) {
        P.slots[t] = P.positions[t] = -1;
        continue;
      }
      while (t >= s_new[b + 1]) {
        ++b;
        block = -1;
      }
      const int p = s_cur[b] + t - s_new[b];
      if (p / COW_PAGE_TOKENS != block) {
        block = p / COW_PAGE_TOKENS;
        page = page_of(b, block);
      }
      P.slots[t] = page * COW_PAGE_TOKENS + p % COW_PAGE_TOKENS;
      P.positions[t] = p;
    }
  }

  // the last block changes what the others may have been reading
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    s_last = atomicInc(reinterpret_cast<unsigned*>(P.ticket), gridDim.x - 1) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!s_last) return;
  for (int b = tid; b < R; b += kResizeThreads) P.lengths[b] = s_target[b];
  if (tid == 0) *P.free_count = count + freed - taken;
  if (mixed) {
    for (int k = tid; k < freed; k += kResizeThreads) {
      const int b = owner_of(s_freed, R, k);
      P.tables[b * P.max_blocks + page_count(s_target[b]) + (k - s_freed[b])] = -1;
    }
  }
}

int64_t max_pieces(int64_t requests, int64_t tokens) {
  const int64_t pages = tokens / COW_PAGE_TOKENS + 2 * requests;
  return tokens < pages ? tokens : pages;
}

}  // namespace

extern "C" {

int64_t cow_pages_plan_words(int64_t requests, int64_t tokens) {
  if (requests < 0 || requests > COW_MAX_REQUESTS || tokens < 0 || tokens >= (int64_t{1} << 31)) return -1;
  return 4 + 4 * max_pieces(requests, tokens) + requests + 1 + 2 * tokens;
}

int cow_pages_resize(const cow_kv_pages* cache, const int32_t* targets, int64_t tokens, int32_t* plan,
                     int64_t plan_words, void* stream) {
  if (!cache || !plan || !aligned16(plan) || !cache->status || !cache->ticket || !cache->free_count ||
      cache->requests < 0 || cache->max_blocks < 0 || cache->pages < 0)
    return COW_ERR_INVALID;
  const int64_t requests = cache->requests, words = cow_pages_plan_words(requests, tokens);
  if (words < 0 || requests * cache->max_blocks >= (1 << 25) || cache->pages >= (1 << 25)) return COW_ERR_UNSUPPORTED;
  if (plan_words < words || (requests > 0 && (!targets || !cache->lengths)) ||
      (requests * cache->max_blocks > 0 && !cache->block_tables) || (cache->pages > 0 && !cache->free_pages))
    return COW_ERR_INVALID;
  const int64_t pieces = max_pieces(requests, tokens);
  int32_t* starts = plan + 4 + 4 * pieces;
  ResizeLaunch P{cache->block_tables, cache->lengths, cache->free_pages, cache->free_count, cache->status,
                 cache->ticket, targets, plan, reinterpret_cast<int4*>(plan + 4), starts, starts + requests + 1,
                 starts + requests + 1 + tokens, cache->max_blocks, static_cast<int32_t>(requests),
                 static_cast<int32_t>(tokens), static_cast<int32_t>(pieces), static_cast<int32_t>(cache->pages)};
  const size_t smem = sizeof(int) * (6 * static_cast<size_t>(requests) + 4);
  if (!resident_blocks(reinterpret_cast<const void*>(cow_pages_resize_kernel), kResizeThreads,
                       sizeof(int) * (6 * COW_MAX_REQUESTS + 4)))
    return COW_ERR_CUDA;
  // a block for each 2,048 tokens of the maps and 2,048 table entries (pages may move without tokens), one for each SM at most
  const int grid = grid_for(tokens + requests * cache->max_blocks, kResizeThreads * kTokensPerThread, 148);
  cow_pages_resize_kernel<<<grid, kResizeThreads, smem, as_stream(stream)>>>(P);
  return launch_status();
}

}  // extern "C"
