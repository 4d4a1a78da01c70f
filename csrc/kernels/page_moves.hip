// Pages of the K/V cache that change their place: copies (a sequence forks, a thread moves) and the compaction of sequences
// whose tokens leave.  Caches are [layers][pages][kv heads][PAGE][row], K and V, with strides between layers, pages and heads;
// a token's row of a head is row_bytes contiguous bytes, a page of a head PAGE rows.
#include "common.h"

namespace {

constexpr int PAGE = 64;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct Cache {   // strides in bytes
  char* p;
  long layer, page, head;
};

// ---- copies ----
// The pairs travel in the launch's own arguments: no copy to the device and no memory to keep until the launch has run.  A
// workgroup takes a page of a head in a layer, 16 bytes a thread, so a token's row of any type is whole pieces.  Bound by memory:
// 203 pages of 8 heads in 8 layers, 400 MB read and as much written, 157 us = 5.1 TB/s (a large copy has 4.9); one page in 32
// layers is a launch of 4 us, behind 8 us of the host's.
constexpr int PAIRS = 256;
struct Pairs {
  int src[PAIRS], dst[PAIRS];
  uint8_t tokens[PAIRS];
};

__global__ __launch_bounds__(256) void copy_pages_kernel(Cache k, Cache v, Pairs pairs, int heads, int layers, int row_bytes) {
  const int h = blockIdx.x % heads, layer = blockIdx.x / heads % layers, i = blockIdx.x / heads / layers;
  const Cache c = blockIdx.y ? v : k;
  const int n = pairs.tokens[i] * row_bytes / 16;
  const long at = layer * c.layer + h * c.head;
  const u32x4* from = (const u32x4*)(c.p + at + pairs.src[i] * c.page);
  u32x4* to = (u32x4*)(c.p + at + pairs.dst[i] * c.page);
  for (int j = threadIdx.x; j < n; j += 256) to[j] = from[j];
}

// ---- compaction ----
struct Sequences {
  const int *tables, *to, *lens;      // tables, to: [n][width]; to null: in place
  const uint8_t* keep;                // [n][places], rows keep_stride apart
  int width, table_stride, to_stride, places, num_pages;
  long keep_stride;
  int* new_lens;
};

__device__ __forceinline__ int length_of(const Sequences& s, int seq) {
  return max(0, min(s.lens[seq], min(s.places, s.width * PAGE)));
}

// A thread holds 16 bytes of each half of a token's row (numbers d and d + 64 of a rotated key meet in one thread), so a
// token takes TPT = row_bytes / 32 threads.
struct Row {
  u32x4 lo, hi;
};

__device__ __forceinline__ Row load_row(const char* p, int half) { return {*(const u32x4*)p, *(const u32x4*)(p + half)}; }
__device__ __forceinline__ void store_row(char* p, int half, const Row& r) {
  *(u32x4*)p = r.lo;
  *(u32x4*)(p + half) = r.hi;
}

// Key numbers i and i + 64, rotated for place `from`, turned on to place `to`: by the angle between the two, whose cosine and
// sine come from the table's of both places in fp32; one rounding to bf16 at the end.
struct Turn {
  float c[8], s[8];
  __device__ __forceinline__ void set(const float* cos_sin, int from, int to, int d) {
    const f32x4* a = (const f32x4*)(cos_sin + ((long)from * 64 + d) * 2);
    const f32x4* b = (const f32x4*)(cos_sin + ((long)to * 64 + d) * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 x = a[i], y = b[i];
      c[2 * i] = fmaf(y[0], x[0], y[1] * x[1]);
      s[2 * i] = fmaf(y[1], x[0], -(y[0] * x[1]));
      c[2 * i + 1] = fmaf(y[2], x[2], y[3] * x[3]);
      s[2 * i + 1] = fmaf(y[3], x[2], -(y[2] * x[3]));
    }
  }
  __device__ __forceinline__ void apply(Row& r) const {
    bf16x8 lo = __builtin_bit_cast(bf16x8, r.lo), hi = __builtin_bit_cast(bf16x8, r.hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = (float)lo[i], y = (float)hi[i];
      lo[i] = f2bf(fmaf(x, c[i], -(y * s[i])));
      hi[i] = f2bf(fmaf(y, c[i], x * s[i]));
    }
    r.lo = __builtin_bit_cast(u32x4, lo);
    r.hi = __builtin_bit_cast(u32x4, hi);
  }
};

// places of `keep` that are set among 8 from p (which need not be aligned)
__device__ __forceinline__ int set_of_8(const uint8_t* p) {
  uint64_t x;
  __builtin_memcpy(&x, p, 8);
  const uint64_t low = 0x7f7f7f7f7f7f7f7full;
  return __popcll((((x & low) + low) | x) & ~low);
}

// Into other pages: a workgroup takes 256 / TPT consecutive places of one sequence, counts the kept ones before them, and
// moves them in the layers and heads of its share (blockIdx.z): the turn's numbers are formed once for all of them.  Places that
// are not kept are not read.  Bound by memory (8 heads, half of the tokens kept): 6 sequences of 8150 places in 8 layers, 0.8 GB
// read and as much written, 331 us = 4.8 TB/s, turned 332; one of 1000 in 32 layers, 131 MB, 30 and 31 us, where one round of
// workgroups has its chain of counting, page numbers, angles, rows and stores.
template <int TPT, bool TURN>
__global__ __launch_bounds__(256) void compact_apart_kernel(Cache k, Cache v, Sequences s, int heads, int layers,
                                                            const float* __restrict__ cos_sin) {
  constexpr int TOK = 256 / TPT, HALF = TPT * 16;
  const int seq = blockIdx.y, tid = threadIdx.x, t = tid / TPT, part = tid % TPT;
  const int len = length_of(s, seq), p0 = blockIdx.x * TOK, place = p0 + t;
  const bool last = p0 + TOK >= len;      // of the sequence's workgroups
  if (p0 >= len && p0 > 0) return;
  const uint8_t* keep = s.keep + seq * s.keep_stride;
  __shared__ int count[4];
  int before = 0;
  for (int j = tid * 8; j < p0; j += 256 * 8) before += set_of_8(keep + j);   // p0 is a multiple of 8
  const bool kept = place < len && keep[place] != 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
  __shared__ int here[4];                                    // kept places of a wavefront
  const unsigned long long set = __ballot(kept && part == 0);   // one lane per place
  const int w = tid >> 6, lane = tid & 63;
  if (lane == 0) {
    count[w] = before;
    here[w] = __popcll(set);
  }
  __syncthreads();
  int to = count[0] + count[1] + count[2] + count[3];
  if (last && blockIdx.z == 0 && tid == 0) s.new_lens[seq] = to + here[0] + here[1] + here[2] + here[3];
  if (!kept) return;
  for (int x = 0; x < w; ++x) to += here[x];
  to += __popcll(set & ((1ull << (lane - part)) - 1));
  const int from_page = s.tables[(long)seq * s.table_stride + place / PAGE], to_page = s.to[(long)seq * s.to_stride + to / PAGE];
  if ((unsigned)from_page >= (unsigned)s.num_pages || (unsigned)to_page >= (unsigned)s.num_pages) return;
  Turn turn;
  const bool turned = TURN && to != place;
  if (turned) turn.set(cos_sin, place, to, part * 8);
  const long inside_from = (long)(place % PAGE) * 2 * HALF + part * 16, inside_to = (long)(to % PAGE) * 2 * HALF + part * 16;
  const int all = heads * layers;
  for (int i = blockIdx.z; i < all; i += gridDim.z) {
    const int h = i % heads, layer = i / heads;
    const char* kf = k.p + layer * k.layer + h * k.head + from_page * k.page + inside_from;
    const char* vf = v.p + layer * v.layer + h * v.head + from_page * v.page + inside_from;
    Row a = load_row(kf, HALF);
    const Row b = load_row(vf, HALF);
    if (turned) turn.apply(a);
    store_row(k.p + layer * k.layer + h * k.head + to_page * k.page + inside_to, HALF, a);
    store_row(v.p + layer * v.layer + h * v.head + to_page * v.page + inside_to, HALF, b);
  }
}

// In place: one workgroup moves all of a sequence's tokens of HEADS heads, a round of 1024 / TPT places after the other.  A place
// n takes the token of a place p >= n: once the workgroup has read a round's places no later read meets what it writes, and the
// next round's reads go out before this one's writes.  1024 threads, since what a CU has in flight is one round: 6 sequences of
// 8150 places in 8 layers (8 heads, half kept), 0.8 GB read and as much written, 356 us = 4.5 TB/s, turned 453; with few
// sequences it is bound by the chain of rounds, some 2.2 us each (one of 1000 in 8 layers 21 us, turned 32, into other pages
// 10 and 11).  Reading `keep`
// two rounds ahead and unrolled rounds gave nothing.
template <int TPT, bool TURN, int HEADS>
__global__ __launch_bounds__(1024) void compact_inside_kernel(Cache k, Cache v, Sequences s, int heads,
                                                              const float* __restrict__ cos_sin) {
  constexpr int TOK = 1024 / TPT, HALF = TPT * 16;
  const int seq = blockIdx.y, h0 = blockIdx.x % (heads / HEADS) * HEADS, layer = blockIdx.x / (heads / HEADS);
  const int tid = threadIdx.x, t = tid / TPT, part = tid % TPT, w = tid >> 6, lane = tid & 63;
  const int len = length_of(s, seq);
  const uint8_t* keep = s.keep + seq * s.keep_stride;
  const int* table = s.tables + (long)seq * s.table_stride;
  char* kp = k.p + layer * k.layer + h0 * k.head + part * 16;
  char* vp = v.p + layer * v.layer + h0 * v.head + part * 16;
  __shared__ int here[2][16];   // kept places of a wavefront, of this round and the one before
  __shared__ int start;
  // the pages: in LDS (a round waits for its places' new pages), those of longer sequences where they are
  constexpr int PAGES = 4096;
  __shared__ int pages[PAGES];
  for (int i = tid; i < min((len + PAGE - 1) / PAGE, PAGES); i += 1024) pages[i] = table[i];
  const auto page_of = [&](int place) {
    const int i = place / PAGE;
    return i < PAGES ? pages[i] : table[i];
  };
  // the places before the first that is not kept stay: rounds begin there
  if (tid == 0) start = len;
  __syncthreads();
  int mine = len;
  for (int p = tid * 8; p < len; p += 1024 * 8) {
    if (p + 8 <= len && set_of_8(keep + p) == 8) continue;
    mine = p;
    break;
  }
  if (mine < len) atomicMin(&start, mine);
  __syncthreads();
  int base = start < len ? start / TOK * TOK : len, side = 0;   // kept places before the round, all of them until here

  bool kept = false, next_kept = false;   // this thread's place of a round, of the next
  const auto look = [&](int p0) { return p0 + t < len && keep[p0 + t] != 0; };
  Row a[HEADS], b[HEADS];
  const auto load = [&](int p0, bool is) {
    const int pg = is ? page_of(p0 + t) : -1;
    if ((unsigned)pg >= (unsigned)s.num_pages) return;
    const long in = (long)((p0 + t) % PAGE) * 2 * HALF;
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      a[h] = load_row(kp + h * k.head + pg * k.page + in, HALF);
      b[h] = load_row(vp + h * v.head + pg * v.page + in, HALF);
    }
  };
  const int p_first = base;
  kept = look(p_first);
  load(p_first, kept);
  for (int p0 = p_first; p0 < len; p0 += TOK, side ^= 1) {
    const int place = p0 + t;
    next_kept = look(p0 + TOK);
    const unsigned long long set = __ballot(kept && part == 0);   // one lane per place
    if (lane == 0) here[side][w] = __popcll(set);
    __syncthreads();
    int to = base + __popcll(set & ((1ull << (lane - part)) - 1));
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const int n = here[side][x];
      base += n;
      if (x < w) to += n;
    }
    const int to_page = kept ? page_of(to) : -1;
    const bool moves = kept && to != place && (unsigned)to_page < (unsigned)s.num_pages
                       && (unsigned)page_of(place) < (unsigned)s.num_pages;
    Turn turn;
    if constexpr (TURN)
      if (moves) turn.set(cos_sin, place, to, part * 8);
    Row x[HEADS], y[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      x[h] = a[h];
      y[h] = b[h];
    }
    // every wavefront's loads have come back before any writes
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    load(p0 + TOK, next_kept);
    if (moves) {
      const long in = (long)(to % PAGE) * 2 * HALF;
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
        if constexpr (TURN) turn.apply(x[h]);
        store_row(kp + h * k.head + to_page * k.page + in, HALF, x[h]);
        store_row(vp + h * v.head + to_page * v.page + in, HALF, y[h]);
      }
    }
    kept = next_kept;
  }
  if (blockIdx.x == 0 && tid == 0) s.new_lens[seq] = base;
}

template <int TPT, bool TURN>
int compact(Cache k, Cache v, const Sequences& s, int n, int heads, int layers, const float* cos_sin, hipStream_t st) {
  if (!s.to) {
    // Two heads in flight per workgroup, once that leaves 192 workgroups (8 heads, half of the tokens kept): six sequences of
    // 8150 places in 8 layers turned 616 -> 453 us, as they are 421 -> 356, six of 1000 75 -> 56 and 57 -> 49, two of 1000 in 32
    // layers 82 -> 64 and 65 -> 56; three of 1000 in 8 would lose, 36 -> 41 and 26 -> 30, one in 32 40 -> 46 and 31 -> 37.
    if (heads % 2 == 0 && heads * layers * n >= 384)
      hipLaunchKernelGGL((compact_inside_kernel<TPT, TURN, 2>), dim3(heads / 2 * layers, n), dim3(1024), 0, st, k, v, s, heads, cos_sin);
    else
      hipLaunchKernelGGL((compact_inside_kernel<TPT, TURN, 1>), dim3(heads * layers, n), dim3(1024), 0, st, k, v, s, heads, cos_sin);
    return (int)hipGetLastError();
  }
  constexpr int TOK = 256 / TPT;
  const int chunks = max(1, (min(s.places, s.width * PAGE) + TOK - 1) / TOK), all = heads * layers;
  // Eight (layer, head) pairs for a workgroup, which counts kept places and forms angles once for them: six sequences of 8150
  // places in 8 layers of 8 heads, half kept, turned 332 us, with one pair each 448, with all 64 349 (as they are 331, 338, 347).  Fewer where
  // there would not be 256 workgroups: one layer of 1000 places 7.6 -> 6.3.
  const int shares = max(max(1, all / 8), min(all, 256 / max(1, chunks * n)));
  hipLaunchKernelGGL((compact_apart_kernel<TPT, TURN>), dim3(chunks, n, shares), dim3(256), 0, st, k, v, s, heads, layers, cos_sin);
  return (int)hipGetLastError();
}

}  // namespace

// Pages src[i] copied to dst[i] (host arrays), the first tokens[i] rows of every head in every layer.  No page may be in dst
// twice or in both, which the caller has checked.  strides: bytes between layers, pages and heads of K, then of V.
P2P_API int p2p_copy_pages(void* k, void* v, const long* strides, int layers, int heads, int num_pages, int row_bytes,
                           const int* src, const int* dst, const int* tokens, int n, hipStream_t stream) {
  if (layers < 1 || heads < 1 || row_bytes < 16 || row_bytes % 16 || n < 0) return (int)hipErrorInvalidValue;
  const Cache ck = {(char*)k, strides[0], strides[1], strides[2]}, cv = {(char*)v, strides[3], strides[4], strides[5]};
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages || tokens[i] < 0 || tokens[i] > PAGE)
      return (int)hipErrorInvalidValue;
  for (int i = 0; i < n;) {
    Pairs pairs;
    int m = 0;
    for (; i < n && m < PAIRS; ++i) {
      if (src[i] == dst[i] || tokens[i] == 0) continue;
      pairs.src[m] = src[i];
      pairs.dst[m] = dst[i];
      pairs.tokens[m++] = (uint8_t)tokens[i];
    }
    if (m == 0) break;
    hipLaunchKernelGGL(copy_pages_kernel, dim3(heads * layers * m, 2), dim3(256), 0, stream, ck, cv, pairs, heads, layers, row_bytes);
    if (int e = (int)hipGetLastError()) return e;
  }
  return 0;
}

// Kept tokens of n sequences to the front of their tables (to null) or of other pages; new_lens[i]: how many.  cos_sin
// (bf16 rows of 128 only): keys turned from their old places to their new ones.
P2P_API int p2p_compact_pages(void* k, void* v, const long* strides, int layers, int heads, int num_pages, int row_bytes,
                              const int* tables, int table_stride, int width, const int* to, int to_stride, const int* lens,
                              const void* keep, long keep_stride, int places, int n, const float* cos_sin, int* new_lens,
                              hipStream_t stream) {
  if (layers < 1 || heads < 1 || n < 1 || width < 0 || places < 0) return (int)hipErrorInvalidValue;
  if (cos_sin && row_bytes != 256) return (int)hipErrorInvalidValue;
  const Cache ck = {(char*)k, strides[0], strides[1], strides[2]}, cv = {(char*)v, strides[3], strides[4], strides[5]};
  const Sequences s = {tables, to, lens, (const uint8_t*)keep, width, table_stride, to_stride, places, num_pages, keep_stride,
                       new_lens};
  switch (row_bytes) {
    case 128: return compact<4, false>(ck, cv, s, n, heads, layers, nullptr, stream);
    case 256:
      return cos_sin ? compact<8, true>(ck, cv, s, n, heads, layers, cos_sin, stream)
                     : compact<8, false>(ck, cv, s, n, heads, layers, nullptr, stream);
    case 512: return compact<16, false>(ck, cv, s, n, heads, layers, nullptr, stream);
  }
  return (int)hipErrorInvalidValue;
}
