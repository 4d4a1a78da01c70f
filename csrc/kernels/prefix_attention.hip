// Attention of query rows whose sequences begin with the same pages of the K/V cache (pages as in paged_attention.hip): the
// shared keys are read once for all rows of a group, every sequence's own keys once for its rows.
//
//   o[r][h] = sum_{j < ctx[r]} softmax_j(scale q[r][h] . k[j]) v[j]
//
// A softmax over keys in parts: part c gives m_c = max of its scores, l_c = sum exp(s - m_c), o_c = sum exp(s - m_c) v, and
// o = sum_c exp(m_c - M) o_c / sum_c exp(m_c - M) l_c with M = max m_c.  So a row's keys may be cut anywhere and each piece
// be done together with other rows that see the same keys.  The host cuts the batch into works (`Work`): query rows of one
// group (or of one sequence) against a range of pages, in `of` parts; the parts' results (fp32) meet in a second launch.
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
  int part, of;        // this is part `part` of `of` equal ones of the pages that some row sees
  int slot;            // and part slot + part of its rows' results
};

__device__ __forceinline__ int kperm(int rho) {  // S^T row rho -> key within the 32 keys (see flash_prefill.hip)
  const int s = rho >> 4, r = rho & 15;
  return 16 * s + 8 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3);
}

// Four wavefronts, each with its own 32 keys at a time against the same 32 (row, head) pairs: S^T = K . Q^T and
// O^T += V^T . P^T in 32x32x16 products, a pair per lane, as in flash_prefill2_kernel.  K and V come by LDS DMA into the
// wavefront's own LDS, the next K while this one's weights are formed, the next V behind the second product; no barrier
// until the four meet at the end.  P is rounded to bf16 for the product (relative 2^-9, as in flash_prefill.hip: what a
// value's weight is off by); scores, maxima, sums and O are fp32.
constexpr int NW = 4, KT = 32, ROWS = 32;

__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefix_attn_kernel(
    const bf16* __restrict__ q, int ldq, const bf16* __restrict__ kc, const bf16* __restrict__ vc, int num_pages,
    const int* __restrict__ bt, int bt_stride, const int* __restrict__ ctx_lens, int max_ctx, const Work* __restrict__ works,
    int n_works, const int* __restrict__ base, int Hkv, int G, float scale_log2, float* __restrict__ part_o, float2* __restrict__ part_ml) {
  __shared__ __attribute__((aligned(16))) bf16 lds[NW][2][KT * HD];   // K and V of every wavefront; its O at the end
  __shared__ float2 sml[NW][ROWS];
  const int b = xcd_remap(blockIdx.x, n_works * Hkv);
  const Work W = works[b / Hkv];
  const int kvh = b % Hkv;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r32 = lane & 31, hh = lane >> 5;
  const int pairs = W.n * G, pair = min(r32, pairs - 1), row = W.row0 + pair / G, head = kvh * G + pair % G;
  const int lim = min(ctx_lens[row], max_ctx);   // keys that this lane's row sees
  int most = lim;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
  most = __builtin_amdgcn_readfirstlane(most);
  const int np = max(0, (min(most, W.page1 * PAGE) + PAGE - 1) / PAGE - W.page0);   // pages that some row sees
  const int first = W.page0 + (int)((long)np * W.part / W.of), end = W.page0 + (int)((long)np * (W.part + 1) / W.of);
  const int last = min(most, end * PAGE) - 1;             // last key
  const int u0 = first * 2 + w, u1 = first < end ? last / KT + 1 : 0;   // units of 32 keys, this wavefront's every fourth

  const size_t page_sz = (size_t)Hkv * PAGE * HD, head_off = (size_t)kvh * PAGE * HD;
  const int* btr = bt + (size_t)W.table * bt_stride;
  const unsigned l0 = __builtin_amdgcn_readfirstlane(ldsp::lds_off(&lds[w][0][0]));
  const int cr = lane >> 4, cp = lane & 15;
  // an instruction takes four rows of 256 bytes; rows past the last key (whatever they hold) are that key's again
  auto copy = [&](const bf16* pool, int u, int page, bool is_v) {
    const bf16* from = pool + (size_t)page * page_sz + head_off + (size_t)(u % 2) * KT * HD;
    const int top = last - u * KT;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = cr + 4 * i;
      ldsp::dma_lds16(from, min(r, top) * (HD * 2) + ((cp ^ (is_v ? 4 * (r & 3) : r & 15)) << 4),
                      l0 + is_v * (KT * HD * 2) + i * 1024);
    }
  };
  auto page_of = [&](int u) { return min(max(btr[min(u, u1 - 1) / 2], 0), num_pages - 1); };

  bf16x8 qf[8];
  {
    const bf16* qp = q + (size_t)row * ldq + (size_t)head * HD + 8 * hh;
#pragma unroll
    for (int s = 0; s < 8; ++s) qf[s] = *reinterpret_cast<const bf16x8_u*>(qp + 16 * s);
  }
#pragma unroll
  for (int s = 0; s < 8; ++s) asm volatile("" : "+v"(qf[s]));   // loaded before the copies are counted
  f32x16 o[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m = -INFINITY, l = 0.f;

  const int krow = kperm(r32), L = lane & 15;
  const bf16* kl = &lds[w][0][krow * HD];
  const bf16* vl = &lds[w][1][(8 * hh + (L >> 2)) * HD + 4 * (L & 1)];
  const int vp = 2 * ((lane >> 4) & 1) + ((L >> 1) & 1);
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4* lds4_t;
  auto read_v = [&](int db, int s2) {   // V^T of numbers 32 db + r32, keys 16 s2 + 8 hh + 0 .. 7
    const bf16* p = vl + 16 * s2 * HD + ((((db ^ (L >> 2)) << 2) | vp) << 3);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(p + 4 * HD));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  if (u0 < u1) {
    int page = page_of(u0);
    copy(kc, u0, page, false);
    copy(vc, u0, page, true);
    page = page_of(u0 + NW);
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
        if (more) copy(kc, u + NW, page, false);
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
        for (int s = 0; s < 8; ++s) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s], qf[s], sc, 0, 0, 0);
      }
      const int k0 = u * KT;
      if (__any(k0 + KT > lim)) {
#pragma unroll
        for (int rr = 0; rr < 16; ++rr)
          if (k0 + 16 * (rr >> 3) + 8 * hh + (rr & 7) >= lim) sc[rr] = -INFINITY;
      }
      float mx = sc[0];
#pragma unroll
      for (int rr = 1; rr < 16; ++rr) mx = fmaxf(mx, sc[rr]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = fmaxf(m, mx);
      const float ms = mn == -INFINITY ? 0.f : mn * scale_log2;    // no key yet: weights 0
      const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * scale_log2);
      m = mn;
      float ps = 0.f;
      bf16x8 pf[2];
#pragma unroll
      for (int rr = 0; rr < 16; ++rr) {
        const float p = __builtin_amdgcn_exp2f(fmaf(sc[rr], scale_log2, -ms));
        ps += p;
        pf[rr >> 3][rr & 7] = f2bf(p);
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
      if (more) copy(vc, u + NW, page, true);
      page = page_of(u + 2 * NW);
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db][s2], pf[s2], o[db], 0, 0, 0);
    }
  }
  l += __shfl_xor(l, 32, 64);
  // the four meet: O of pair r32 as rows of 512 bytes, 16-byte piece p at p ^ r32
  float* so = reinterpret_cast<float*>(&lds[w][0][0]);
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {   // registers 4 g4 ..: numbers 32 db + 8 g4 + 4 hh + 0 .. 3
      const int piece = 8 * db + 2 * g4 + hh;
      *reinterpret_cast<f32x4*>(so + r32 * HD + ((piece ^ r32) << 2)) =
          f32x4{o[db][4 * g4], o[db][4 * g4 + 1], o[db][4 * g4 + 2], o[db][4 * g4 + 3]};
    }
  if (hh == 0) sml[w][r32] = make_float2(m == -INFINITY ? m : m * scale_log2, l);
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(lds);
#pragma unroll
  for (int i = 0; i < ROWS * 32 / (NW * 64); ++i) {
    const int at = tid + i * NW * 64, p = at >> 5, piece = at & 31;
    if (p >= pairs) break;
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < NW; ++x) M = fmaxf(M, sml[x][p].x);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float2 ml = sml[x][p];
      const float e = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);
      sum += *reinterpret_cast<const f32x4*>(all + x * (KT * HD) + p * HD + ((piece ^ p) << 2)) * e;
      den = fmaf(e, ml.y, den);
    }
    const int r = W.row0 + p / G;
    const size_t to = ((size_t)(base[r] + W.slot + W.part) * Hkv + kvh) * G + p % G;
    *reinterpret_cast<f32x4*>(part_o + to * HD + 4 * piece) = sum;
    if (piece == 0) part_ml[to] = make_float2(M, den);
  }
}

// One (row, head) pair of a wavefront, key by key in fp32: what a row sees of values that are not finite.  Products of tiles
// give 0 * inf = nan to rows of the tile that do not see the value.
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
    const float p = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - mn);
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
  acc[0] /= l;
  acc[1] /= l;
}

// The parts of a row: a wavefront per (row, head), two numbers per lane.
__global__ __launch_bounds__(256) void prefix_combine_kernel(
    const bf16* __restrict__ q, int ldq, const bf16* __restrict__ kc, const bf16* __restrict__ vc, int num_pages,
    const int* __restrict__ bt, int bt_stride, const int* __restrict__ ctx_lens, int max_ctx, const int* __restrict__ base,
    const int* __restrict__ tables, int R, int Hkv, int G, float scale_log2, const float* __restrict__ part_o,
    const float2* __restrict__ part_ml, bf16* __restrict__ out, int ldo) {
  const int Hq = Hkv * G, lane = threadIdx.x & 63;
  const int i = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (i >= R * Hq) return;
  const int r = i / Hq, h = i % Hq;
  const int b0 = base[r], n = base[r + 1] - b0;
  float M = -INFINITY;
  for (int c = lane; c < n; c += 64) M = fmaxf(M, part_ml[(size_t)(b0 + c) * Hq + h].x);
  M = wave_max(M);
  float acc[2] = {0.f, 0.f}, den = 0.f;
  for (int c0 = 0; c0 < n; c0 += 64) {
    float e = 0.f;
    if (c0 + lane < n) {
      const float2 ml = part_ml[(size_t)(b0 + c0 + lane) * Hq + h];
      e = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);
      den = fmaf(e, ml.y, den);
    }
    const int nc = min(64, n - c0);
#pragma unroll 8
    for (int c = 0; c < nc; ++c) {
      const float2 v = *reinterpret_cast<const float2*>(part_o + ((size_t)(b0 + c0 + c) * Hq + h) * HD + 2 * lane);
      const float ec = __shfl(e, c, 64);
      acc[0] = fmaf(ec, v.x, acc[0]);
      acc[1] = fmaf(ec, v.y, acc[1]);
    }
  }
  den = wave_sum(den);
  if (M == -INFINITY && !(den != den)) {
    acc[0] = acc[1] = 0.f;    // no key
  } else {
    acc[0] /= den;
    acc[1] /= den;
    if (__any(!(fabsf(acc[0]) < INFINITY) || !(fabsf(acc[1]) < INFINITY)))
      exact_pair(q + (size_t)r * ldq + (size_t)h * HD, kc, vc, bt + (size_t)tables[r] * bt_stride, num_pages,
                 (size_t)Hkv * PAGE * HD, (size_t)(h / G) * PAGE * HD, min(ctx_lens[r], max_ctx), scale_log2, lane, acc);
  }
  bf16* op = out + (size_t)r * ldo + (size_t)h * HD + 2 * lane;
  op[0] = f2bf(acc[0]);
  op[1] = f2bf(acc[1]);
}

}  // namespace

// works: int32 [n_works, 8] (Work); base: int32 [R + 1], the parts of the rows before; tables: int32 [R], the rows' block
// tables; part_o, part_ml: base[R] * Hq * (128 | 2) floats.  Every part of every row belongs to one work.
P2P_API int p2p_prefix_attention(const void* q, int ldq, const void* k_cache, const void* v_cache, int num_pages,
                                 const int* block_tables, int bt_stride, const int* ctx_lens, int max_ctx, const int* works,
                                 int n_works, const int* base, const int* tables, int R, int Hq, int Hkv, int head_dim, float scale,
                                 void* out, int ldo, float* part_o, float* part_ml, hipStream_t stream) {
  if (head_dim != HD || Hkv <= 0 || Hq % Hkv || Hq / Hkv > ROWS || R <= 0 || n_works <= 0) return (int)hipErrorInvalidValue;
  const float sl2 = scale * 1.4426950408889634f;
  const int G = Hq / Hkv;
  hipLaunchKernelGGL(prefix_attn_kernel, dim3(n_works * Hkv), dim3(NW * 64), 0, stream, (const bf16*)q, ldq,
                     (const bf16*)k_cache, (const bf16*)v_cache, num_pages, block_tables, bt_stride, ctx_lens, max_ctx,
                     (const Work*)works, n_works, base, Hkv, G, sl2, part_o, (float2*)part_ml);
  if (int e = (int)hipGetLastError()) return e;
  hipLaunchKernelGGL(prefix_combine_kernel, dim3((R * Hq + 3) / 4), dim3(256), 0, stream, (const bf16*)q, ldq,
                     (const bf16*)k_cache, (const bf16*)v_cache, num_pages, block_tables, bt_stride, ctx_lens, max_ctx, base,
                     tables, R, Hkv, G, sl2, part_o, (const float2*)part_ml, (bf16*)out, ldo);
  P2P_CHECK_LAUNCH();
}
