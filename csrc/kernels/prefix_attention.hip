// Attention of query rows whose sequences begin with the same pages of the K/V cache (pages as in paged_attention.hip): the
// shared keys are read once for all rows of a group, every sequence's own keys once for its rows.
//
//   o[r][h] = sum_{j < ctx[r]} softmax_j(scale q[r][h] . k[j]) v[j]
//
// A softmax over keys in parts: part c gives m_c = max of its scores, l_c = sum exp(s - m_c), o_c = sum exp(s - m_c) v, and
// o = sum_c exp(m_c - M) o_c / sum_c exp(m_c - M) l_c with M = max m_c.  So a row's keys may be cut anywhere and each piece
// be done together with other rows that see the same keys.  The host cuts the batch into works (`Work`): query rows of one
// group (or of one sequence) against a range of pages, in `of` parts; the parts' results (fp32) meet in a second launch.
//
// What it takes, calls one after the other: 2 rows behind 256 tokens 7 us (the host 8), 19 behind 2048 13 and 41 on one kv head
// 15, of which the second launch is 3: chains of loads of some 0.7 us each (work, page numbers, keys, values) and the launches.
// 704 prompt rows behind 1536 tokens 34 us, 64 rows of 64 heads behind 32768 108 us: chains between the products, see the tiles.
#include "common.h"
#include "lds_pipe.h"

namespace {

constexpr int PAGE = 64, HD = 128;
typedef bf16x8 bf16x8_u __attribute__((aligned(2)));   // rows of q and out of any alignment
typedef bf16x4 bf16x4_u __attribute__((aligned(2)));

struct Work {
  int row0, n;         // query rows
  int table;           // block-table row whose pages they read
  int page0, page1;    // pages
  int part, of;        // this is part `part` of `of` equal ones of the pages that some row sees (of 0: these are the part's pages)
  int slot;            // and part slot + part of its rows' results
};

__device__ __forceinline__ int kperm(int rho) {  // S^T row rho -> key within the 32 keys (see flash_prefill.hip)
  const int s = rho >> 4, r = rho & 15;
  return 16 * s + 8 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3);
}

constexpr int ROWS = 32;
constexpr int PG = PAGE * HD;                    // numbers of a page's K (V)

struct Args {
  const bf16 *q, *kc, *vc;
  const int *bt, *ctx_lens, *base;
  float* part_o;
  float2* part_ml;
  bf16* out;
  int ldq, ldo, num_pages, bt_stride, max_ctx, Hkv, G;
  int even;              // parts of every row, where they are equally many (1: the results themselves), else 0
  float scale_log2;
};

// A workgroup's share of a work: pages first .. end - 1, of whose keys the last that some row sees is `last`.
struct Share {
  int first, end, last;
};
__device__ __forceinline__ Share share_of(const Work& W, int most) {
  if (W.of == 0) return {W.page0, W.page1, W.page1 * PAGE - 1};   // (known before the context lengths have come)
  const int np = max(0, (min(most, W.page1 * PAGE) + PAGE - 1) / PAGE - W.page0);
  const int first = W.page0 + (int)((long)np * W.part / W.of), end = W.page0 + (int)((long)np * (W.part + 1) / W.of);
  return {first, end, min(most, end * PAGE) - 1};
}
__device__ __forceinline__ int most_of(const Args& A, const Work& W, int lane) {   // keys that some row sees
  int most = 0;
  for (int r = lane; r < W.n; r += 64) most = max(most, min(A.ctx_lens[W.row0 + r], A.max_ctx));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
  return __builtin_amdgcn_readfirstlane(most);
}
__device__ __forceinline__ int least_of(int lim) {   // of the wavefront's 32 rows
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lim = min(lim, __shfl_xor(lim, o, 64));
  return __builtin_amdgcn_readfirstlane(lim);
}
// A work's page numbers, through scalar loads: a vector load's wait would be one for the copies in flight, too.
struct Pages {
  const __attribute__((address_space(4))) int* row;
  int num_pages;
  __device__ __forceinline__ Pages(const Args& A, const Work& W)
      : row((const __attribute__((address_space(4))) int*)(uintptr_t)(A.bt + (size_t)W.table * A.bt_stride)), num_pages(A.num_pages) {}
  __device__ __forceinline__ int entry(int at) const { return row[at]; }
  __device__ __forceinline__ int page(int entry) const { return min(max(entry, 0), num_pages - 1); }
  __device__ __forceinline__ int operator()(int at) const { return page(entry(at)); }
};

__device__ __forceinline__ float max_of_halves(float x) {   // of lanes i and i + 32
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// Q^T operand of a lane's (row, head) pair: k-step s covers numbers 16 s .. 16 s + 15, lane half hh has 8 hh .. 8 hh + 7
__device__ __forceinline__ void load_q(const Args& A, int row, int head, int hh, bf16x8 (&qf)[8]) {
  const bf16* qp = A.q + (size_t)row * A.ldq + (size_t)head * HD + 8 * hh;
#pragma unroll
  for (int s = 0; s < 8; ++s) qf[s] = *reinterpret_cast<const bf16x8_u*>(qp + 16 * s);
}
// Waits for them (and with them for every copy so far): the first copies go out before, and from here on waits are counted
__device__ __forceinline__ void have_q(bf16x8 (&qf)[8]) {
#pragma unroll
  for (int s = 0; s < 8; ++s) asm volatile("" : "+v"(qf[s]));
}

// A lane's O (numbers 32 db + 8 g4 + 4 hh + 0 .. 3 of pair r32) as rows of 512 bytes in LDS, 16-byte piece p at p ^ r32
__device__ __forceinline__ void put_rows(float* so, const f32x16 (&o)[4], int r32, int hh) {
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      *reinterpret_cast<f32x4*>(so + r32 * HD + (((8 * db + 2 * g4 + hh) ^ r32) << 2)) =
          f32x4{o[db][4 * g4], o[db][4 * g4 + 1], o[db][4 * g4 + 2], o[db][4 * g4 + 3]};
}
__device__ __forceinline__ f32x4 get_row(const float* so, int pair, int piece) {
  return *reinterpret_cast<const f32x4*>(so + pair * HD + ((piece ^ pair) << 2));
}

// Where a pair's numbers go: into out where its row has one part, else into the parts' outputs
__device__ __forceinline__ long place_of(const Args& A, const Work& W, int kvh, int pair) {
  const int row = W.row0 + pair / A.G, head = kvh * A.G + pair % A.G;
  if (A.even == 1) return (long)row * A.ldo + head * HD;
  const int before = A.even ? row * A.even : A.base[row];
  return ((long)(before + W.slot + W.part) * A.Hkv * A.G + head) * HD;
}

// One (row, head) pair of a wavefront, key by key in fp32: what a row sees of values that are not finite (products of tiles
// give 0 * inf = nan to rows of the tile that do not see the value), and a row without a weight: 0 where it has no key, nan
// where all of its keys' scores are -inf.  Weights are 2^-32 of what they are elsewhere: sums of finite values, up to 2^32 of the
// largest, stay finite, and what falls below 2^-126 is 2^-94 of the largest weight at most.
__device__ void exact_pair(const bf16* qp, const bf16* kc, const bf16* vc, const int* btr, int num_pages, size_t page_sz,
                           size_t head_off, int ctx, float scale_log2, int lane, float (&acc)[2]) {
  float m = -INFINITY, l = 0.f;
  acc[0] = acc[1] = 0.f;
  for (int k0 = 0; k0 < ctx; k0 += PAGE) {
    const size_t page = (size_t)min(max(btr[k0 / PAGE], 0), num_pages - 1) * page_sz + head_off;
    float s = -INFINITY;
    if (k0 + lane < ctx) {
      const bf16* kp = kc + page + (size_t)lane * HD;
      s = 0.f;
      for (int d = 0; d < HD; ++d) s = fmaf((float)kp[d], (float)qp[d], s);
      s *= scale_log2;
    }
    const float mn = fmaxf(m, wave_max(s));
    const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    const float p = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - mn) * 0x1p-32f;
    m = mn;
    l = fmaf(l, alpha, wave_sum(p));
    acc[0] *= alpha;
    acc[1] *= alpha;
    const int n = min(PAGE, ctx - k0);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl(p, j, 64);
      const bf16x2 v = *reinterpret_cast<const bf16x2*>(vc + page + (size_t)j * HD + 2 * lane);
      acc[0] = fmaf(pj, (float)v[0], acc[0]);
      acc[1] = fmaf(pj, (float)v[1], acc[1]);
    }
  }
  acc[0] = ctx > 0 ? acc[0] / l : 0.f;
  acc[1] = ctx > 0 ? acc[1] / l : 0.f;
}
// the same for row r's head h, from the row's block table `btr`
__device__ void exact_pair(const Args& A, const int* btr, int r, int h, int lane, float (&acc)[2]) {
  exact_pair(A.q + (size_t)r * A.ldq + (size_t)h * HD, A.kc, A.vc, btr, A.num_pages, (size_t)A.Hkv * PG, (size_t)(h / A.G) * PG,
             min(A.ctx_lens[r], A.max_ctx), A.scale_log2, lane, acc);
}
__device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) < INFINITY); }

// A pair's result from its only part: lane r32 has numbers 4 r32 ..  True: it has to be done again.
__device__ __forceinline__ bool put_result(const Args& A, long at, f32x4 sum, float den, bool sees, int r32) {
  const float by = 1.f / den;
  bf16x4 y;
  bool bad = den == 0.f && sees;   // (no score above -inf)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = den == 0.f ? 0.f : sum[i] * by;   // (whatever the values of others are)
    bad |= not_finite(x);
    y[i] = f2bf(x);
  }
  *reinterpret_cast<bf16x4_u*>(A.out + at + 4 * r32) = y;
  return bad;
}
__device__ void put_exact(const Args& A, const Work& W, int kvh, int pair, int lane) {
  const int r = W.row0 + pair / A.G, h = kvh * A.G + pair % A.G;
  float acc[2];
  exact_pair(A, A.bt + (size_t)W.table * A.bt_stride, r, h, lane, acc);
  bf16* op = A.out + (size_t)r * A.ldo + (size_t)h * HD + 2 * lane;
  op[0] = f2bf(acc[0]);
  op[1] = f2bf(acc[1]);
}


typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds4_t;
// eight keys of a V^T operand from rows of 256 bytes, 16-byte piece p of row r at p ^ 4 (r & 3): `p` is this lane's place
__device__ __forceinline__ bf16x8 read_v8(const bf16* p) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)p);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(p + 4 * HD));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---- up to 128 pairs ----
// Four wavefronts have 32 pairs each and share the pages; with KG = 2 four more have the same pairs and every other page (two
// pages of a workgroup on its way, one result of them: half the results of two workgroups).  K and V of a page come by LDS DMA,
// two stages each, and a page's exponentials run between the products of the page before with V, as in flash_prefill2_kernel
// (whose layouts these are).  P is rounded to bf16 for the product (relative 2^-8 at most: what a value's weight is off by);
// scores, maxima, sums and O are fp32.
//
// A wavefront reads a page's K and V from LDS, 32 KB, for 32 matrix instructions of 32 cycles: two workgroups on a CU have 2050
// cycles of either for a page each, and take 4300 to 4900 (2.0 to 2.3 us at 2.13 GHz, the clock under this load), also where
// all pages are one that the caches hold: a wavefront's chain of maxima, exponentials and waits at a page's start, which one
// other wavefront on its SIMD does not cover.  64 rows of 64 heads behind 32768 tokens, 69 GFLOP: 81 us, of which launch, first
// loads and 34 MB of results 12.
// Three stages of K, a barrier of its own for V, copies spread between the products, LDS reads three pairs ahead and both
// products interleaved (which spills) gave nothing.
// 128 pairs, since a wavefront's registers hold 32 (O 64, Q 64, S and P 64) and four are a CU's quarters: with 32 pairs for a
// workgroup 241 us, 129 then with 128 (with the rows' own tokens and the second launch).
template <int KG>
__device__ __forceinline__ void tile_role(const Args& A, const Work& W, int kvh, bf16* lds_all, float2* sml, int wave, int lane) {
  constexpr int CW = 4, CP = 16 / CW;                       // wavefronts that copy a page together, copies of each
  const int w = wave % CW, kg = wave / CW;                  // pairs 32 w .., pages first + kg, first + kg + KG, ..
  bf16* lds = lds_all + kg * (4 * PG);                      // K, K, V, V
  const int r32 = lane & 31, hh = lane >> 5;
  const Pages pages(A, W);
  const Share S = share_of(W, W.of ? most_of(A, W, lane) : 0);
  const int pairs = W.n * A.G, mine = w * 32 + r32, pair = min(mine, pairs - 1), row = W.row0 + pair / A.G;
  const int lim = min(min(A.ctx_lens[row], A.max_ctx), S.end * PAGE), least = least_of(lim);
  long to = S.first < S.end ? 0 : mine < pairs ? place_of(A, W, kvh, mine) : -1;
  f32x16 o[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  if (S.first < S.end) {
    const size_t page_sz = (size_t)A.Hkv * PG, head_off = (size_t)kvh * PG;
    // an instruction takes four rows of 256 bytes; rows past the last key (whatever they hold) are that key's again
    const unsigned l0 = __builtin_amdgcn_readfirstlane(ldsp::lds_off(lds)) + w * 1024;
    const int cr = 4 * w + (lane >> 4), cp = lane & 15;
    unsigned koff[CP], voff[CP];
#pragma unroll
    for (int i = 0; i < CP; ++i) {
      const int r = cr + 4 * CW * i;
      koff[i] = r * (HD * 2) + ((cp ^ (r & 15)) << 4);
      voff[i] = r * (HD * 2) + ((cp ^ (4 * (r & 3))) << 4);
    }
    auto copy = [&](const bf16* pool, int kt, int page, unsigned dst, const unsigned (&off)[CP]) {
      const bf16* from = pool + (size_t)page * page_sz + head_off;
      const int top = S.last - min(kt, S.end - 1) * PAGE;
      if (top >= PAGE - 1) {
#pragma unroll
        for (int i = 0; i < CP; ++i) ldsp::dma_lds16(from, off[i], dst + i * CW * 1024);
      } else {
#pragma unroll
        for (int i = 0; i < CP; ++i)
          ldsp::dma_lds16(from, off[i] - max(cr + 4 * CW * i - top, 0) * (HD * 2), dst + i * CW * 1024);
      }
    };
    // (a group's last turn may be a page past the end: that is the last page again, of which it sees no key)
    const int turns = (S.end - S.first + KG - 1) / KG;
    auto entry_of = [&](int t) { return pages.entry(min(S.first + KG * t + kg, S.end - 1)); };
    auto copy_k = [&](int t, int page) { copy(A.kc, S.first + KG * t + kg, page, l0 + (t & 1) * (PG * 2), koff); };
    auto copy_v = [&](int t, int page) { copy(A.vc, S.first + KG * t + kg, page, l0 + (2 + (t & 1)) * (PG * 2), voff); };
    int p0 = pages.page(entry_of(0)), p1 = entry_of(1);   // this turn's page, the next one's entry in the block table
    int flip = PG * 2;                      // from this turn's stage to the other
    bf16x8 qf[8];
    load_q(A, row, kvh * A.G + pair % A.G, hh, qf);
    copy_k(0, p0);
    copy_v(0, p0);
    if (turns > 1) copy_k(1, pages.page(p1));

    // places of this lane in a stage: K rows kperm(r32) (and 32 further), V as read_v8 takes it
    const int krow = kperm(r32), L = lane & 15;
    int kat[8], vat[4];   // (in bytes)
#pragma unroll
    for (int s = 0; s < 8; ++s) kat[s] = (krow * HD + (((2 * s + hh) ^ (krow & 15)) << 3)) * 2;
#pragma unroll
    for (int db = 0; db < 4; ++db)
      vat[db] = (2 * PG + (8 * hh + (L >> 2)) * HD + 4 * (L & 1) +
                 ((((db ^ (L >> 2)) << 2) | (2 * ((lane >> 4) & 1) + ((L >> 1) & 1))) << 3)) * 2;
    const char* at_lds = reinterpret_cast<const char*>(lds);
    f32x16 sc[2];
    bf16x8 pf[2][2];   // P^T of the page before
    // O^T += V^T . P^T of the page before in eight pairs of products; LDS reads go out a pair ahead, and between them runs `work`
    auto second_product = [&](auto&& work) {
      bf16x8 vf[2][2];
      auto read_v2 = [&](int j) {   // numbers 32 (j / 2) .., keys 32 (j & 1) + 16 i ..
#pragma unroll
        for (int i = 0; i < 2; ++i) vf[j & 1][i] = read_v8(reinterpret_cast<const bf16*>(at_lds + vat[j >> 1]) + (32 * (j & 1) + 16 * i) * HD);
      };
      read_v2(0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < 7) read_v2(j + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          o[j >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[j & 1][i], pf[j & 1][i], o[j >> 1], 0, 0, 0);
          work(2 * j + i);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int db = 0; db < 4; ++db) vat[db] += flip;   // (first_product has turned it round once more)
    };
    // S^T = K . Q^T of turn t's page, two halves of 32 keys; the copies of its V and of the next K go out first
    auto first_product = [&](int t) {
      // K of this page and V of the one before have landed; every wave is past the last page's K and the V before it
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (t > 0) {
        copy_v(t, p0);
        if (t + 1 < turns) copy_k(t + 1, pages.page(p1));
      }
      p0 = pages.page(p1);
      bf16x8 kf[2][2];
      auto read_k2 = [&](int s) {
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) kf[s & 1][kh] = *reinterpret_cast<const bf16x8*>(at_lds + kat[s] + 32 * kh * HD * 2);
      };
      read_k2(0);
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        if (s < 7) read_k2(s + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
          sc[kh] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s & 1][kh], qf[s], s == 0 ? f32x16{} : sc[kh], 0, 0, 0);
      }
#pragma unroll
      for (int s = 0; s < 8; ++s) kat[s] += flip;
      flip = -flip;
      // Keys of register rr of half kh: 16 (rr >> 3) + 8 hh + (rr & 7)
      const int k0 = (S.first + KG * t + kg) * PAGE, left = lim - k0 - 8 * hh;
      if (k0 + PAGE > least) {
        asm volatile("");   // (a branch, not selects on every page)
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
#pragma unroll
          for (int rr = 0; rr < 16; ++rr)
            if (32 * kh + 16 * (rr >> 3) + (rr & 7) >= left) sc[kh][rr] = -INFINITY;
      }
    };
    float alpha, mc, ps;
    // The maxima.  O and l are rescaled only when some row's grew by more than 2^8 (wave-uniform): until then weights stay
    // below 2^8, as exact in bf16 as below 1.
    auto maxima = [&] {
      constexpr float RESCALE_THR = 8.f;
      float mx = fmaxf(sc[0][0], sc[1][0]), my = fmaxf(sc[0][1], sc[1][1]);
#pragma unroll
      for (int rr = 2; rr < 16; rr += 2) {
        mx = fmaxf(fmaxf(mx, sc[0][rr]), sc[1][rr]);
        my = fmaxf(fmaxf(my, sc[0][rr + 1]), sc[1][rr + 1]);
      }
      mx = max_of_halves(fmaxf(mx, my));
      const bool rescale = __any((mx - m) * A.scale_log2 > RESCALE_THR);
      if (rescale) {
        const float mn = fmaxf(m, mx);
        alpha = mn == m ? 1.f : __builtin_amdgcn_exp2f((m - mn) * A.scale_log2);   // (no key yet: -inf both)
        m = mn;
        l *= alpha;
      }
      mc = m == -INFINITY ? 0.f : m * A.scale_log2;
      ps = 0.f;
      int again = __builtin_amdgcn_readfirstlane(rescale);
      asm volatile("" : "+s"(again));   // (one copy of what follows, not one for each side of the branch)
      return again;
    };
    unsigned pn[4][4];   // this page's P^T
    auto exps = [&](int j) {   // two of 32
      const int kh = j >> 3, rr = (j & 7) * 2;
      const float x = __builtin_amdgcn_exp2f(fmaf(sc[kh][rr], A.scale_log2, -mc));
      const float y = __builtin_amdgcn_exp2f(fmaf(sc[kh][rr + 1], A.scale_log2, -mc));
      const bf16x2 xy = {f2bf(x), f2bf(y)}, ones = {(bf16)1.f, (bf16)1.f};
      ps = __builtin_amdgcn_fdot2_f32_bf16(xy, ones, ps, false);   // (of the weights as they go into the product)
      pn[2 * kh + (rr >> 3)][(rr & 7) / 2] = __builtin_bit_cast(unsigned, xy);
      // (formed here, between the products, not where they are used)
      asm volatile("" : "+v"(pn[2 * kh + (rr >> 3)][(rr & 7) / 2]), "+v"(ps));
    };
    auto take = [&](int t) {
      // (the entry for the turn after the next: on its way while the copies are waited for, not while LDS reads are counted)
      __builtin_amdgcn_sched_barrier(0);
      p1 = entry_of(t + 2);
      __builtin_amdgcn_sched_barrier(0);
      l += ps;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        pf[i >> 1][i & 1] = __builtin_bit_cast(bf16x8, u32x4{pn[i][0], pn[i][1], pn[i][2], pn[i][3]});
      }
    };
    to = mine < pairs ? place_of(A, W, kvh, mine) : -1;   // (while the copies are on their way)
    asm volatile("" : "+v"(to));
    have_q(qf);
    first_product(0);
    maxima();
#pragma unroll
    for (int j = 0; j < 16; ++j) exps(j);
    take(0);
    for (int t = 1; t < turns; ++t) {
      first_product(t);
      const int rescale = maxima();
      second_product(exps);
      take(t);
      if (rescale) {   // (O has the page before by now, which the old maximum scaled)
#pragma unroll
        for (int db = 0; db < 4; ++db) o[db] *= alpha;
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    second_product([](int) {});
    __syncthreads();
  }
  l += __shfl_xor(l, 32, 64);
  m = m == -INFINITY ? m : m * A.scale_log2;
  const bool whole = A.even == 1;
  if (!whole && (KG == 1 || S.first >= S.end) && kg == 0 && hh == 0 && to >= 0) A.part_ml[to / HD] = make_float2(m, l);
  if (!whole && S.first >= S.end) return;   // a part of no page has its maximum only
  // the wavefront's rows to LDS and from there in whole rows, of both page groups: 32 / KG pairs for a wavefront
  const unsigned sees = (unsigned)__ballot(lim > 0);   // pairs that see a key
  float* so = reinterpret_cast<float*>(lds_all);
  put_rows(so + wave * (32 * HD), o, r32, hh);
  if constexpr (KG > 1) {
    if (hh == 0) sml[wave * 32 + r32] = make_float2(m, l);
    __syncthreads();
  } else {
    __builtin_amdgcn_wave_barrier();
  }
  unsigned bad = 0;
#pragma unroll
  for (int i = 0; i < 16 / KG; ++i) {
    const int p = kg * (32 / KG) + 2 * i + hh;
    const long at = __shfl(to, p, 64);
    f32x4 sum = get_row(so + w * (32 * HD), p, r32);
    float den = KG == 1 && whole ? __shfl(l, p, 64) : 0.f;
    if constexpr (KG > 1) {
      const float2 a = sml[w * 32 + p], b = sml[(CW + w) * 32 + p];
      const float M = fmaxf(a.x, b.x);
      const float ea = a.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(a.x - M);
      const float eb = b.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(b.x - M);
      sum = sum * ea + get_row(so + (CW + w) * (32 * HD), p, r32) * eb;
      den = fmaf(ea, a.y, eb * b.y);
      if (!whole && at >= 0 && r32 == 0) A.part_ml[at / HD] = make_float2(M, den);
    }
    if (at < 0) continue;
    if (whole) bad |= (unsigned)put_result(A, at, sum, den, sees >> p & 1, r32) << i;
    else *reinterpret_cast<f32x4*>(A.part_o + at + 4 * r32) = sum;
  }
  if (__builtin_expect(__any(bad), 0)) {
#pragma unroll 1
    for (int i = 0; i < 32 / KG; ++i)
      if ((__ballot(bad >> (i / 2) & 1) >> (32 * (i & 1))) & 0xffffffffull)
        put_exact(A, W, kvh, w * 32 + kg * (32 / KG) + i, lane);
  }
}

// ---- up to 32 pairs ----
// NW wavefronts, each with its own 32 keys at a time against the same pairs.  K and V come by LDS DMA into the wavefront's
// own LDS, the next K while this one's weights are formed, the next V behind the second product; no barrier until they meet at
// the end.  For up to 32 pairs, where of a tile's four wavefronts three had nothing to do: so they take different keys instead,
// and a CU has four streams of loads, which is what few rows are bound by.  2 rows behind 1024 tokens, 6 MB, 8.2 us.
constexpr int KT = 32;

template <int NW>
__device__ __forceinline__ void few_role(const Args& A, const Work& W, int kvh, bf16* lds_all, float2* sml, int w, int lane) {
  bf16* lds = lds_all + w * (2 * KT * HD);   // K and V; O at the end
  const int r32 = lane & 31, hh = lane >> 5;
  const Pages pages(A, W);
  const int pairs = W.n * A.G, pair = min(r32, pairs - 1), row = W.row0 + pair / A.G;
  const int lim = min(A.ctx_lens[row], A.max_ctx), least = least_of(lim);
  const Share S = share_of(W, W.of ? most_of(A, W, lane) : 0);
  const int u0 = S.first * 2 + w, u1 = S.first < S.end ? S.last / KT + 1 : 0;   // units of 32 keys, every NW-th for this wavefront

  const size_t page_sz = (size_t)A.Hkv * PG, head_off = (size_t)kvh * PG;
  const unsigned l0 = __builtin_amdgcn_readfirstlane(ldsp::lds_off(lds));
  const int cr = lane >> 4, cp = lane & 15;
  auto copy = [&](const bf16* pool, int u, int page, bool is_v) {
    const bf16* from = pool + (size_t)page * page_sz + head_off + (size_t)(u % 2) * KT * HD;
    const int top = S.last - u * KT;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = cr + 4 * i;
      ldsp::dma_lds16(from, min(r, top) * (HD * 2) + ((cp ^ (is_v ? 4 * (r & 3) : r & 15)) << 4),
                      l0 + is_v * (KT * HD * 2) + i * 1024);
    }
  };
  auto page_of = [&](int u) { return pages(min(u, u1 - 1) / 2); };

  bf16x8 qf[8];
  load_q(A, row, kvh * A.G + pair % A.G, hh, qf);
  f32x16 o[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m = -INFINITY, l = 0.f;

  const int krow = kperm(r32), L = lane & 15;
  const bf16* kl = lds + krow * HD;
  const bf16* vl = lds + KT * HD + (8 * hh + (L >> 2)) * HD + 4 * (L & 1);
  const int vp = 2 * ((lane >> 4) & 1) + ((L >> 1) & 1);
  auto read_v = [&](int db, int s2) {   // V^T of numbers 32 db + r32, keys 16 s2 + 8 hh + 0 .. 7
    return read_v8(vl + 16 * s2 * HD + ((((db ^ (L >> 2)) << 2) | vp) << 3));
  };

  if (u0 < u1) {
    int page = page_of(u0);
    copy(A.kc, u0, page, false);
    copy(A.vc, u0, page, true);
    page = page_of(u0 + NW);
    have_q(qf);
    for (int u = u0; u < u1; u += NW) {
      const bool more = u + NW < u1;
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");    // K (V's eight copies follow)
      __builtin_amdgcn_wave_barrier();
      f32x16 sc;
      {
        bf16x8 kf[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) kf[s] = *reinterpret_cast<const bf16x8*>(kl + (((2 * s + hh) ^ (krow & 15)) << 3));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int s = 0; s < 8; ++s) asm volatile("" : "+v"(kf[s]));
        if (more) copy(A.kc, u + NW, page, false);
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
        for (int s = 0; s < 8; ++s) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s], qf[s], sc, 0, 0, 0);
      }
      const int left = lim - u * KT - 8 * hh;
      if (u * KT + KT > least) {
        asm volatile("");
#pragma unroll
        for (int rr = 0; rr < 16; ++rr)
          if (16 * (rr >> 3) + (rr & 7) >= left) sc[rr] = -INFINITY;
      }
      float mx = sc[0];
#pragma unroll
      for (int rr = 1; rr < 16; ++rr) mx = fmaxf(mx, sc[rr]);
      mx = max_of_halves(mx);
      const float mn = fmaxf(m, mx);
      const float ms = mn == -INFINITY ? 0.f : mn * A.scale_log2;    // no key yet: weights 0
      const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * A.scale_log2);
      m = mn;
      float ps = 0.f;
      bf16x8 pf[2];
#pragma unroll
      for (int rr = 0; rr < 16; rr += 2) {   // (rounded for the product and summed so, as in a tile)
        const bf16x2 xy = {f2bf(__builtin_amdgcn_exp2f(fmaf(sc[rr], A.scale_log2, -ms))),
                           f2bf(__builtin_amdgcn_exp2f(fmaf(sc[rr + 1], A.scale_log2, -ms)))},
                     ones = {(bf16)1.f, (bf16)1.f};
        ps = __builtin_amdgcn_fdot2_f32_bf16(xy, ones, ps, false);
        pf[rr >> 3][rr & 7] = xy[0];
        pf[rr >> 3][(rr & 7) + 1] = xy[1];
      }
      l = fmaf(l, alpha, ps);
#pragma unroll
      for (int db = 0; db < 4; ++db) o[db] *= alpha;
      if (more) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      bf16x8 vf[4][2];
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) vf[db][s2] = read_v(db, s2);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) asm volatile("" : "+v"(vf[db][s2]));
      if (more) copy(A.vc, u + NW, page, true);
      page = page_of(u + 2 * NW);
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db][s2], pf[s2], o[db], 0, 0, 0);
    }
  }
  l += __shfl_xor(l, 32, 64);
  const long to = r32 < pairs ? place_of(A, W, kvh, r32) : -1;
  const bool whole = A.even == 1;
  if (!whole && S.first >= S.end) {   // a part of no page has its maximum only
    if (w == 0 && hh == 0 && to >= 0) A.part_ml[to / HD] = make_float2(-INFINITY, 0.f);
    return;
  }
  put_rows(reinterpret_cast<float*>(lds), o, r32, hh);   // (in this wavefront's own K and V)
  if (hh == 0) sml[w * ROWS + r32] = make_float2(m == -INFINITY ? m : m * A.scale_log2, l);
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(lds_all);
  const unsigned sees = (unsigned)__ballot(lim > 0);   // pairs that see a key
  unsigned bad = 0;
#pragma unroll
  for (int i = 0; i < ROWS * 32 / (NW * 64); ++i) {
    const int p = 2 * (NW * i + w) + hh;
    const long at = __shfl(to, p, 64);
    float2 ml[NW];
    float M = -INFINITY, den = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      ml[x] = sml[x * ROWS + p];
      M = fmaxf(M, ml[x].x);
    }
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float e = ml[x].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[x].x - M);
      den = fmaf(e, ml[x].y, den);
      sum += get_row(all + x * (KT * HD), p, r32) * e;
    }
    if (at < 0) continue;
    if (whole) {
      bad |= (unsigned)put_result(A, at, sum, den, sees >> p & 1, r32) << i;
      continue;
    }
    *reinterpret_cast<f32x4*>(A.part_o + at + 4 * r32) = sum;
    if (r32 == 0) A.part_ml[at / HD] = make_float2(M, den);
  }
  if (__builtin_expect(__any(bad), 0)) {
#pragma unroll 1
    for (int i = 0; i < 2 * (ROWS * 32 / (NW * 64)); ++i)
      if ((__ballot(bad >> (i / 2) & 1) >> (32 * (i & 1))) & 0xffffffffull)
        put_exact(A, W, kvh, 2 * (NW * (i / 2) + w) + (i & 1), lane);
  }
}

template <int NW, bool TILES>   // TILES: some work has more than 32 pairs
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefix_attn_kernel(
    Args A, const Work* __restrict__ works) {
  constexpr int KG = NW / 4;
  static_assert(NW * 2 * KT * HD == KG * 4 * PG, "both roles in the same LDS");
  __shared__ __attribute__((aligned(16))) bf16 lds[KG * 4 * PG];
  __shared__ float2 sml[NW * 32];   // maxima and sums of every wavefront's pairs
  // heads first: with 8 kv heads an XCD has one of them, and its L2 that head's pages for all tiles
  const int b = blockIdx.x;
  const Work W = works[b / A.Hkv];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (TILES && W.n * A.G > ROWS) tile_role<KG>(A, W, b % A.Hkv, lds, sml, w, lane);
  else few_role<NW>(A, W, b % A.Hkv, lds, sml, w, lane);
}

// The parts of a (row, head) pair: GROUPS half wavefronts, four numbers per lane, each with every GROUPS-th part.  A group has
// the statistics and outputs of eight parts in flight together, what they weigh is known when they have come; groups meet in LDS.
// Bound by memory where there is much (4096 pairs of 17 parts, 36 MB, 9.5 us = 3.8 TB/s), else by its launch: 608 pairs 3 us.
template <int GROUPS>
__global__ __launch_bounds__(256) void prefix_combine_kernel(Args A, const int* __restrict__ tables, int R) {
  const int Hq = A.Hkv * A.G, lane = threadIdx.x & 63, r32 = lane & 31, g = GROUPS == 1 ? 0 : threadIdx.x >> 5;
  const int pair0 = GROUPS == 1 ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x, pair = min(pair0, R * Hq - 1);
  const int r = pair / Hq, h = pair % Hq;
  const int b0 = A.even ? r * A.even : A.base[r], n = A.even ? A.even : A.base[r + 1] - b0;
  const float2* ml = A.part_ml + (size_t)b0 * Hq + h;
  const float* po = A.part_o + ((size_t)b0 * Hq + h) * HD + 4 * r32;
  float M = -INFINITY, den = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = g; c0 < n; c0 += 8 * GROUPS) {
    float2 st[8];
    f32x4 o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const size_t c = (size_t)min(c0 + j * GROUPS, n - 1) * Hq;
      st[j] = ml[c];
      o[j] = *reinterpret_cast<const f32x4*>(po + c * HD);
    }
    float m = M;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = c0 + j * GROUPS < n ? fmaxf(m, st[j].x) : m;
    const float alpha = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - m);
    M = m;
    den *= alpha;
    acc *= alpha;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (c0 + j * GROUPS >= n) break;
      const float e = st[j].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[j].x - m);
      den = fmaf(e, st[j].y, den);
      // (of no weight: nothing may be written there)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = e == 0.f ? acc[i] : fmaf(e, o[j][i], acc[i]);
    }
  }
  if constexpr (GROUPS > 1) {
    __shared__ f32x4 so[GROUPS][32];
    __shared__ float2 sml[GROUPS];
    so[g][r32] = acc;
    if (r32 == 0) sml[g] = make_float2(M, den);
    __syncthreads();
    if (threadIdx.x >= 64) return;
    M = -INFINITY;
#pragma unroll
    for (int x = 0; x < GROUPS; ++x) M = fmaxf(M, sml[x].x);
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
    den = 0.f;
#pragma unroll
    for (int x = 0; x < GROUPS; ++x) {
      const float2 s = sml[x];
      const float e = s.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s.x - M);
      den = fmaf(e, s.y, den);
      acc += so[x][r32] * e;
    }
  }
  const float by = den == 0.f ? 0.f : 1.f / den;   // (0: no key, or none of a score above -inf)
  bf16x4 y;
  bool bad = den == 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = acc[i] * by;
    bad |= not_finite(x);
    y[i] = f2bf(x);
  }
  if (pair0 < R * Hq && (GROUPS == 1 || g == 0))
    *reinterpret_cast<bf16x4_u*>(A.out + (size_t)r * A.ldo + (size_t)h * HD + 4 * r32) = y;
  const unsigned long long again = __ballot(bad);
  if (again) {
    for (int x = 0; x < (GROUPS == 1 ? 2 : 1); ++x) {
      if (!(again >> (32 * x) & 0xffffffffull)) continue;
      const int rx = __shfl(r, 32 * x, 64), hx = __shfl(h, 32 * x, 64);
      float two[2];
      exact_pair(A, A.bt + (size_t)tables[rx] * A.bt_stride, rx, hx, lane, two);
      bf16* op = A.out + (size_t)rx * A.ldo + (size_t)hx * HD + 2 * lane;
      op[0] = f2bf(two[0]);
      op[1] = f2bf(two[1]);
    }
  }
}

}  // namespace

// What a plan hands to its calls (host memory).
struct PrefixPlan {
  const int *works;       // int32 [n_works, 8] (Work); every part of every row belongs to one
  const int *base;        // int32 [R + 1], the parts of the rows before
  const int *tables;      // int32 [R], the rows' block tables
  int n_works, waves, tiles, R, parts, even, Hq, Hkv, head_dim, max_ctx;   // tiles: some work has more than 32 pairs; even:
};                                                                         // the parts of every row, or 0

// workspace: parts * Hq * (128 + 2) floats, outputs and then maxima and sums.
P2P_API int p2p_prefix_attention(const PrefixPlan* plan, const void* q, int ldq, const void* k_cache, const void* v_cache,
                                 int num_pages, const int* block_tables, int bt_stride, const int* ctx_lens, float scale, void* out,
                                 int ldo, float* workspace, hipStream_t stream) {
  const PrefixPlan& P = *plan;
  const int Hq = P.Hq, Hkv = P.Hkv, R = P.R, even = P.even;
  if (P.head_dim != HD || Hkv <= 0 || Hq % Hkv || Hq / Hkv > ROWS || R <= 0 || P.n_works <= 0 || (P.waves != 4 && P.waves != 8))
    return (int)hipErrorInvalidValue;
  const float sl2 = scale * 1.4426950408889634f;
  const int G = Hq / Hkv;
  const Args A = {(const bf16*)q, (const bf16*)k_cache, (const bf16*)v_cache, block_tables, ctx_lens, P.base, workspace,
                  (float2*)(workspace + (size_t)P.parts * Hq * HD), (bf16*)out, ldq, ldo, num_pages, bt_stride, P.max_ctx, Hkv, G,
                  even, sl2};
  const auto kernel = P.waves == 8 ? (P.tiles ? prefix_attn_kernel<8, true> : prefix_attn_kernel<8, false>)
                                   : (P.tiles ? prefix_attn_kernel<4, true> : prefix_attn_kernel<4, false>);
  hipLaunchKernelGGL(kernel, dim3(P.n_works * Hkv), dim3(P.waves * 64), 0, stream, A, (const Work*)P.works);
  if (int e = (int)hipGetLastError()) return e;
  if (even == 1) return 0;
  // A workgroup for each pair where pairs are few, a half wavefront where they fill the chip.  64 pairs of 8 parts 12.8 -> 11.0 us
  // with the parts' own time, of 24 15.9 -> 9.2; 608 of 8 22.2 -> 20.6, 2048 of 10 23.6 -> 22.6 (of 2 80.0 -> 81.3); 4096 of 10
  // 29.1 and 29.5, 8192 of 10 54.5 and 57.3.
  if (P.parts > 3 * R && R * Hq <= 2048)
    hipLaunchKernelGGL(prefix_combine_kernel<8>, dim3(R * Hq), dim3(256), 0, stream, A, P.tables, R);
  else
    hipLaunchKernelGGL(prefix_combine_kernel<1>, dim3((R * Hq + 7) / 8), dim3(256), 0, stream, A, P.tables, R);
  P2P_CHECK_LAUNCH();
}
