// The walk for few sequences (deltanet_chunk.cu): a block takes 32 columns of a
// head's S, four warps 16 of them.  Each of the four holds a quarter of dk of S and
// forms R and d of 16 of a chunk's tokens, so a chunk's products and sums are
// done by eight warps, at the price of three exchanges through shared memory:
// the quarters' parts of S^T k, R, and d.  Four more warps form the outputs
// behind them and copy the chunks to come.
//
// Bound by the chain of those exchanges: 2.9 us a chunk of dk = 128, 2.3 of dk = 64
// (one head, slope from 2048 to 6144 tokens), with the tensor pipe 51 % and the
// issue slots 37 % busy.  A warp per 16 columns (the walk for many sequences) takes
// 5.0 and 3.6 there.
#pragma once

#include "deltanet_chunk_parts.cuh"

namespace qfn {
namespace {

constexpr int kQuadCols = 32;            // state columns of a block
template <int DK>
constexpr int kQuadStages = DK == 128 ? 2 : 3;   // chunks of what the recurrence reads: as many as fit
constexpr int kQuadOutStages = 2;        // chunks of what only the outputs read
constexpr int kQuadThreads = 12 * 32;    // 8 warps of the recurrence, 4 of the outputs and the copies

template <int DK>
struct QuadStage {
  unsigned char k[C * DK * 2];
  unsigned char t[3 * kTermBytes];
  float f[kFactors];
  unsigned char v[C * kQuadCols * 2];
};
template <int DK>
struct QuadOutStage {
  unsigned char q[C * DK * 2], p[kPBytes];
};

// Fragments travel as 16 bytes per lane and term.
template <int DK>
struct QuadSmem {
  QuadStage<DK> stage[kQuadStages<DK>];
  QuadOutStage<DK> out_stage[kQuadOutStages];
  uint4 s[2][2][4][DK / 64][2][32];   // S [buffer][columns][quarter of dk][k tile][term][lane]
  uint4 d[2][2][4][2][32];            // d [buffer][columns][token block][term][lane]
  float4 x[2][4][3][2][32];           // partial S^T k [columns][quarter][block - quarter - 1][tile][lane]
  uint4 rx[2][4][3][32];              // R [columns][token block][term][lane]
  uint4 dx[2][4][3][32];              // weighted d, likewise
  int bad[2][2][16];                  // [buffer][columns][column] first token whose R or d is not finite, or C
  uint64_t full[kQuadStages<DK>], empty[kQuadStages<DK>], out_full[kQuadOutStages], out_empty[kQuadOutStages];
  int length[kSorted], seq;
  uint64_t s_full[2][2], d_full[2][2], out_done[2][2];   // [buffer][columns]
};

__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// The four warps of 16 columns.
__device__ __forceinline__ void quad_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, 128;" ::"r"(id + 1) : "memory");
}

__device__ __forceinline__ uint4 as_uint4(const uint32_t (&r)[4]) { return make_uint4(r[0], r[1], r[2], r[3]); }
__device__ __forceinline__ void from_uint4(uint32_t (&r)[4], uint4 v) { r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w; }

// The output warps of 16 columns take blocks of 16 tokens so that their triangular products take
// the same time: 0 and 3 to one, 1 and 2 to the other.
__device__ __forceinline__ int block_of(int half, int i) { return half ? 1 + i : 3 * i; }

// A block's values of a lane's columns g (first token bad0) and g + 8 (bad1) from those tokens on become NaN.
__device__ __forceinline__ void spoil_block(float* d, int block, int bad0, int bad1) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int tok = block * 16 + i * 8 + 2 * (threadIdx.x & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (tok + (j & 1) >= (j < 2 ? bad0 : bad1)) d[i * 4 + j] = CUDART_NAN_F;
  }
}

template <int DK>
__global__ void __launch_bounds__(kQuadThreads, 1) dn_walk_quad_kernel(const DnRows a, const Plan plan, const Work work,
                                                               int64_t slot0, int64_t slot1, bool vec) {
  extern __shared__ __align__(1024) unsigned char raw[];
  QuadSmem<DK>& sm = *reinterpret_cast<QuadSmem<DK>*>(raw);
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int cb = a.dv / kQuadCols;
  const int c0 = static_cast<int>(blockIdx.x % cb) * kQuadCols;
  const int h = static_cast<int>(blockIdx.x / cb % a.heads);
  if (tid == 0) {
    for (int i = 0; i < kQuadStages<DK>; ++i) {
      mbar_init(&sm.full[i], 129);   // the bulk copies' bytes, 128 lanes' copies of v
      mbar_init(&sm.empty[i], 12);
    }
    for (int i = 0; i < kQuadOutStages; ++i) {
      mbar_init(&sm.out_full[i], 1);
      mbar_init(&sm.out_empty[i], 4);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sm.s_full[0][0] + i, 4);
      mbar_init(&sm.d_full[0][0] + i, 4);
      mbar_init(&sm.out_done[0][0] + i, 2);
    }
    fence_mbar_init();
  }
  pdl_wait();
  const Part part = choose(plan, blockIdx.x / cb / a.heads, slot0, slot1, sm.length, &sm.seq);
  if (part.none(slot1)) return;
  const int64_t seq = part.seq, begin = part.begin, len = part.len, base = part.base, first = part.first, last = part.last;
  const bool ok = part.ok;
  const float* s_from = first > 0 ? a.s_out : a.s_in;
  const int64_t s_at = (seq * a.heads + h) * DK * static_cast<int64_t>(a.dv) + c0;

  if (w < 8) {
    // ---- the recurrence: columns grp * 16 .. + 15; a warp holds a quarter of dk of S and forms R and d of
    // 16 tokens.  The two column groups share the schedulers and do not wait for each other, so one's sums
    // and barriers run under the other's products; the quarters run the other way in the second group,
    // since block 3 has four times block 0's products in T R.
    constexpr int NT = DK / 32, KT = DK / 64;
    const int grp = w >> 2, qd = grp ? 3 - (w & 3) : w & 3, d0 = qd * (DK / 4);
    const float* src = s_from ? s_from + s_at + grp * 16 + g : nullptr;
    float S[NT][4];   // S^T: rows are columns g and g + 8, columns are dk
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int64_t r = static_cast<int64_t>(d0 + i * 8 + 2 * t) * a.dv;
      S[i][0] = src ? src[r] : 0.f;
      S[i][1] = src ? src[r + a.dv] : 0.f;
      S[i][2] = src ? src[r + 8] : 0.f;
      S[i][3] = src ? src[r + a.dv + 8] : 0.f;
    }
    if (!ok) {
#pragma unroll
      for (int i = 0; i < NT; ++i) S[i][0] = S[i][1] = S[i][2] = S[i][3] = CUDART_NAN_F;
    }
    float acc[8][4], vb[2][4];   // this quarter's part of S^T k, blocks qd, qd + 1, .. (mod 4); beta v of the block
    uint32_t kx[KT][4][4];       // k's fragments of the chunk that comes next
    auto load_keys = [&](uint32_t n) {
      wait(&sm.full[n % kQuadStages<DK>], (n / kQuadStages<DK>) & 1);
      const uint32_t kb = smem_u32(sm.stage[n % kQuadStages<DK>].k);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          ldsm4(kx[kt][b], kb + swz<DK * 2>(((qd + b) & 3) * 16 + (lane & 7) + ((lane >> 4) << 3),
                                            d0 / 8 + kt * 2 + ((lane >> 3) & 1)));
    };
    // S's terms times the keys of chunk n; the first two terms go to the warps of the outputs too.  What chunk
    // n's R needs besides comes behind the products.
    auto times_keys = [&](uint32_t n) {
      const uint32_t bf = n & 1;
      const QuadStage<DK>& sn = sm.stage[n % kQuadStages<DK>];
      uint32_t f[KT][3][4];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) frag_split(S[2 * kt], S[2 * kt + 1], f[kt]);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int term = 0; term < 3; ++term)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if (kt == 0 && term == 0) {
              mma_first(acc[2 * b], f[kt][term], kx[kt][b][0], kx[kt][b][1]);
              mma_first(acc[2 * b + 1], f[kt][term], kx[kt][b][2], kx[kt][b][3]);
            } else {
              mma_add(acc[2 * b], f[kt][term], kx[kt][b][0], kx[kt][b][1]);
              mma_add(acc[2 * b + 1], f[kt][term], kx[kt][b][2], kx[kt][b][3]);
            }
          }
      if (n >= 2) wait(&sm.out_done[bf][grp], ((n >> 1) + 1) & 1);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int term = 0; term < 2; ++term) sm.s[bf][grp][qd][kt][term][lane] = as_uint4(f[kt][term]);
      if (qd == 0 && lane < 16) sm.bad[bf][grp][lane] = C;
      warp_arrive(&sm.s_full[bf][grp]);
      uint32_t v[4];   // (columns 0-7 | 8-15) x (tokens 0-7), then tokens 8-15, transposed
      ldsm4t(v, smem_u32(sn.v) + swz<64>(qd * 16 + (lane & 7) + ((lane >> 4) << 3), grp * 2 + ((lane >> 3) & 1)));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 fb = *reinterpret_cast<const float2*>(&sn.f[kFB + qd * 16 + j * 8 + 2 * t]);
        vb[j][0] = fb.x * __uint_as_float(v[2 * j] << 16);
        vb[j][1] = fb.y * __uint_as_float(v[2 * j] & 0xffff0000u);
        vb[j][2] = fb.x * __uint_as_float(v[2 * j + 1] << 16);
        vb[j][3] = fb.y * __uint_as_float(v[2 * j + 1] & 0xffff0000u);
      }
    };
    if (first < last) {
      load_keys(0);
      times_keys(0);
    }
    for (int64_t ci = first; ci < last; ++ci) {
      const uint32_t it = static_cast<uint32_t>(ci - first), st = it % kQuadStages<DK>, buf = it & 1;
      QuadStage<DK>& sg = sm.stage[st];
      const uint32_t kb = smem_u32(sg.k), tb = smem_u32(sg.t) + lane * 16;
      const bool more = ci + 1 < last;
      // the quarters' parts meet, each in the warp of its token block
#pragma unroll
      for (int b = 1; b < 4; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          sm.x[grp][qd][b - 1][j][lane] = make_float4(acc[2 * b + j][0], acc[2 * b + j][1], acc[2 * b + j][2], acc[2 * b + j][3]);
      quad_sync(grp);
      float R[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 o1 = sm.x[grp][(qd + 1) & 3][2][j][lane];
        const float4 o2 = sm.x[grp][(qd + 2) & 3][1][j][lane];
        const float4 o3 = sm.x[grp][(qd + 3) & 3][0][j][lane];
        const float2 fa = *reinterpret_cast<const float2*>(&sg.f[kFA + qd * 16 + j * 8 + 2 * t]);
        R[j][0] = fmaf(fa.x, (acc[j][0] + o1.x) + (o2.x + o3.x), vb[j][0]);
        R[j][1] = fmaf(fa.y, (acc[j][1] + o1.y) + (o2.y + o3.y), vb[j][1]);
        R[j][2] = fmaf(fa.x, (acc[j][2] + o1.z) + (o2.z + o3.z), vb[j][2]);
        R[j][3] = fmaf(fa.y, (acc[j][3] + o1.w) + (o2.w + o3.w), vb[j][3]);
      }
      // A token's infinity or NaN may not reach the tokens before it through T's and P's zeros: it is taken out
      // here and put back into d from that token on.
      auto take_out = [&](float (&x)[2][4]) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!(fabsf(x[i][j]) < CUDART_INF_F)) {
              atomicMin(&sm.bad[buf][grp][g + (j >> 1) * 8], qd * 16 + i * 8 + 2 * t + (j & 1));
              x[i][j] = 0.f;
            }
      };
      if (any_not_finite(R)) take_out(R);
      uint32_t r[3][4];
      frag_split(R[0], R[1], r);
#pragma unroll
      for (int term = 0; term < 3; ++term) sm.rx[grp][qd][term][lane] = as_uint4(r[term]);
      // d = T R of this block, R's blocks qd, qd - 1, .., 0; the products' sums by their size: p[0] of the first
      // terms, p[1] 2^-8 and p[2] 2^-16 of it
      float p[3][2][4];
      auto times_t = [&](const uint32_t (&x)[3][4], int src, bool fresh) {
        uint32_t y[3][4];
#pragma unroll
        for (int term = 0; term < 3; ++term) ldsm4(y[term], tb + term * kTermBytes + tri_block(qd, src));
#pragma unroll
        for (int sum = 0; sum < 3; ++sum)
#pragma unroll
          for (int i = 0; i <= sum; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (fresh && i == 0) mma_first(p[sum][j], x[i], y[sum - i][2 * j], y[sum - i][2 * j + 1]);
              else mma_add(p[sum][j], x[i], y[sum - i][2 * j], y[sum - i][2 * j + 1]);
            }
      };
      times_t(r, qd, true);
      quad_sync(grp);
#pragma unroll
      for (int j = 1; j < 4; ++j)
        if (j <= qd) {
          uint32_t x[3][4];
#pragma unroll
          for (int term = 0; term < 3; ++term) from_uint4(x[term], sm.rx[grp][qd - j][term][lane]);
          times_t(x, qd - j, false);
        }
      // k^T's fragments for the state's update
      uint32_t kt_[4][NT / 2][4];
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int np = 0; np < NT / 2; ++np)
          ldsm4t(kt_[b][np], kb + swz<DK * 2>(((qd + b) & 3) * 16 + (lane & 15), d0 / 8 + np * 2 + (lane >> 4)));
      const int bad0 = sm.bad[buf][grp][g], bad1 = sm.bad[buf][grp][g + 8];
      const bool any_bad = __any_sync(0xffffffffu, bad0 < C || bad1 < C);
      uint32_t wd[3][4];   // d, weighted for the state
      float od[2][4];      // d for the outputs
      {
        float d[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) od[i][j] = p[0][i][j] + (p[1][i][j] + p[2][i][j]);
        if (any_bad) spoil_block(&od[0][0], qd, bad0, bad1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 fw = *reinterpret_cast<const float2*>(&sg.f[kFW + qd * 16 + i * 8 + 2 * t]);
          d[i][0] = od[i][0] * fw.x;
          d[i][1] = od[i][1] * fw.y;
          d[i][2] = od[i][2] * fw.x;
          d[i][3] = od[i][3] * fw.y;
        }
        frag_split(d[0], d[1], wd);
#pragma unroll
        for (int term = 0; term < 3; ++term) sm.dx[grp][qd][term][lane] = as_uint4(wd[term]);
      }
      // S = e^G64 S + d k^T for this quarter of dk
      float u[NT][4];
      auto times_k = [&](const uint32_t (&x)[3][4], int b) {
#pragma unroll
        for (int term = 0; term < 3; ++term)
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            const uint32_t(&y)[4] = kt_[b][np];
            if (b == 0 && term == 0) {
              mma_first(u[2 * np], x[term], y[0], y[1]);
              mma_first(u[2 * np + 1], x[term], y[2], y[3]);
            } else {
              mma_add(u[2 * np], x[term], y[0], y[1]);
              mma_add(u[2 * np + 1], x[term], y[2], y[3]);
            }
          }
      };
      times_k(wd, 0);
      quad_sync(grp);
#pragma unroll
      for (int b = 1; b < 4; ++b) {
        uint32_t x[3][4];
#pragma unroll
        for (int term = 0; term < 3; ++term) from_uint4(x[term], sm.dx[grp][(qd + b) & 3][term][lane]);
        times_k(x, b);
      }
      // d for the outputs of this chunk, under the state's products; a d that overflowed is bad for them, too
      if (any_not_finite(od)) take_out(od);
      {
        uint32_t o[2][4];
        frag_split(od[0], od[1], o);
#pragma unroll
        for (int term = 0; term < 2; ++term) sm.d[buf][grp][qd][term][lane] = as_uint4(o[term]);
      }
      warp_arrive(&sm.d_full[buf][grp]);
      const float keep = sg.f[kFEnd];
      if (more) load_keys(it + 1);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) S[i][j] = fmaf(S[i][j], keep, u[i][j]);
      warp_arrive(&sm.empty[st]);
      if (more) times_keys(it + 1);
    }
    float* dst = a.s_out + s_at + grp * 16 + g;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int64_t r = static_cast<int64_t>(d0 + i * 8 + 2 * t) * a.dv;
      dst[r] = S[i][0];
      dst[r + a.dv] = S[i][1];
      dst[r + 8] = S[i][2];
      dst[r + a.dv + 8] = S[i][3];
    }
  } else {
    // ---- the outputs: columns grp * 16 .. + 15, half of the token blocks per warp; and the copies
    constexpr int KT = DK / 64;
    const int grp = (w - 8) >> 1, half = w & 1, hl = tid - 8 * 32, key_heads = a.heads / a.ratio;
    const uint32_t n = static_cast<uint32_t>(max(last - first, static_cast<int64_t>(0)));
    asm volatile("fence.proxy.async.global;" ::: "memory");   // the other kernel's stores, before bulk copies of them
    auto head_at = [&](uint32_t it) {
      return work.heads + ((base + first + it - slot0) * a.heads + h) * static_cast<int64_t>(kHeadBytes);
    };
    auto keys_at = [&](uint32_t it) {
      return work.kq + ((base + first + it - slot0) * key_heads + h / a.ratio) * (2 * C * DK * 2);
    };
    // chunk `it` of what the recurrence reads, its stage being free
    auto copy_in = [&](uint32_t it) {
      QuadStage<DK>& sg = sm.stage[it % kQuadStages<DK>];
      uint64_t* bar = &sm.full[it % kQuadStages<DK>];
      const int64_t t0 = begin + (first + it) * C;
      const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
      if (hl == 0) {
        mbar_arrive_expect_tx(bar, C * DK * 2 + kRecBytes);
        bulk_g2s(sg.k, keys_at(it), C * DK * 2, bar);
        bulk_g2s(sg.t, head_at(it), kRecBytes, bar);
      }
      __syncwarp();
      const uint16_t* v = a.v + t0 * a.v_row + h * a.v_head + c0;
#pragma unroll
      for (int i = 0; i < C * kQuadCols * 2 / 16 / 128; ++i) {
        const int r = i * 32 + (hl >> 2), ch = hl & 3;
        const uint32_t dst = smem_u32(sg.v) + swz<64>(r, ch);
        const uint16_t* src = v + (r < cnt ? r * a.v_row + ch * 8 : 0);
        if (vec) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(r < cnt ? 16 : 0)
                       : "memory");
        } else {
          uint32_t x[4] = {0, 0, 0, 0};
          if (r < cnt)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = src[2 * j] | static_cast<uint32_t>(src[2 * j + 1]) << 16;
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                       : "memory");
        }
      }
      if (vec)
        asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
      else
        mbar_arrive(bar);
    };
    // chunk `it` of what only the outputs read
    auto copy_out_operands = [&](uint32_t it) {
      QuadOutStage<DK>& og = sm.out_stage[it % kQuadOutStages];
      uint64_t* bar = &sm.out_full[it % kQuadOutStages];
      if (hl == 0) {
        mbar_arrive_expect_tx(bar, C * DK * 2 + kPBytes);
        bulk_g2s(og.q, keys_at(it) + C * DK * 2, C * DK * 2, bar);
        bulk_g2s(og.p, head_at(it) + kRecBytes, kPBytes, bar);
      }
      __syncwarp();
    };
    for (uint32_t i = 0; i < n && i < kQuadStages<DK>; ++i) copy_in(i);
    for (uint32_t i = 0; i < n && i < kQuadOutStages; ++i) copy_out_operands(i);
    for (uint32_t it = 0; it < n; ++it) {
      const uint32_t st = it % kQuadStages<DK>, so = it % kQuadOutStages, buf = it & 1;
      QuadStage<DK>& sg = sm.stage[st];
      QuadOutStage<DK>& og = sm.out_stage[so];
      const int64_t t0 = begin + (first + it) * C;
      const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
      wait(&sm.full[st], (it / kQuadStages<DK>) & 1);
      wait(&sm.out_full[so], (it / kQuadOutStages) & 1);
      wait(&sm.s_full[buf][grp], (it >> 1) & 1);
      const uint32_t qb = smem_u32(og.q), pb = smem_u32(og.p) + lane * 16;
      float o[4][4];   // o^T: rows are columns g and g + 8, tiles of 8 tokens
#pragma unroll
      for (int kt = 0; kt < DK / 16; ++kt) {
        uint32_t x[2][4];
#pragma unroll
        for (int term = 0; term < 2; ++term) from_uint4(x[term], sm.s[buf][grp][kt / KT][kt % KT][term][lane]);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t y[4];
          ldsm4(y, qb + swz<DK * 2>(block_of(half, b) * 16 + (lane & 7) + ((lane >> 4) << 3), kt * 2 + ((lane >> 3) & 1)));
#pragma unroll
          for (int term = 0; term < 2; ++term) {
            if (kt == 0 && term == 0) {
              mma_first(o[2 * b], x[term], y[0], y[1]);
              mma_first(o[2 * b + 1], x[term], y[2], y[3]);
            } else {
              mma_add(o[2 * b], x[term], y[0], y[1]);
              mma_add(o[2 * b + 1], x[term], y[2], y[3]);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = *reinterpret_cast<const float2*>(&sg.f[kFQ + block_of(half, i >> 1) * 16 + (i & 1) * 8 + 2 * t]);
        o[i][0] *= f.x;
        o[i][1] *= f.y;
        o[i][2] *= f.x;
        o[i][3] *= f.y;
      }
      wait(&sm.d_full[buf][grp], (it >> 1) & 1);
#pragma unroll
      for (int bj = 0; bj < 4; ++bj) {
        uint32_t x[2][4];
#pragma unroll
        for (int term = 0; term < 2; ++term) from_uint4(x[term], sm.d[buf][grp][bj][term][lane]);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int bi = block_of(half, b);
          if (bj > bi) continue;
          uint32_t y[2][4];
#pragma unroll
          for (int term = 0; term < 2; ++term) ldsm4(y[term], pb + term * kTermBytes + tri_block(bi, bj));
#pragma unroll
          for (int j = 0; j < 2; ++j) mma_add(o[2 * b + j], x[1], y[0][2 * j], y[0][2 * j + 1]);
#pragma unroll
          for (int j = 0; j < 2; ++j) mma_add(o[2 * b + j], x[0], y[1][2 * j], y[1][2 * j + 1]);
#pragma unroll
          for (int j = 0; j < 2; ++j) mma_add(o[2 * b + j], x[0], y[0][2 * j], y[0][2 * j + 1]);
        }
      }
      {
        const int bad0 = sm.bad[buf][grp][g], bad1 = sm.bad[buf][grp][g + 8];
        if (__any_sync(0xffffffffu, bad0 < C || bad1 < C)) {
          spoil_block(&o[0][0], block_of(half, 0), bad0, bad1);
          spoil_block(&o[2][0], block_of(half, 1), bad0, bad1);
        }
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.out_done[buf][grp]);
        mbar_arrive(&sm.empty[st]);
        mbar_arrive(&sm.out_empty[so]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = block_of(half, i >> 1) * 16 + (i & 1) * 8 + g;   // after the transposition a row is a token
        uint16_t* dst = a.out + ((t0 + tok) * a.heads + h) * a.dv + c0 + grp * 16 + 2 * t;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const __nv_bfloat162 b2 = __floats2bfloat162_rn(o[i][2 * r], o[i][2 * r + 1]);
          const uint32_t y = transpose8x8(*reinterpret_cast<const uint32_t*>(&b2));
          if (tok < cnt) *reinterpret_cast<uint32_t*>(dst + 8 * r) = y;
        }
      }
      if (it + kQuadOutStages < n) {
        wait(&sm.out_empty[so], (it / kQuadOutStages) & 1);
        copy_out_operands(it + kQuadOutStages);
      }
      if (it + kQuadStages<DK> < n) {
        wait(&sm.empty[st], (it / kQuadStages<DK>) & 1);
        copy_in(it + kQuadStages<DK>);
      }
    }
    // nothing of these warps may still be on its way when the block ends
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
}

}  // namespace
}  // namespace qfn
