// The walk for many sequences (deltanet_chunk.cu): a block takes 64 or 128
// columns of a head's S, a warp 16 of them on its own.
//
// No exchange and no barrier in a chunk, so a chunk takes longer than in the quads'
// walk but a block holds two to four times the columns.  Four prompts of 2048
// tokens, 32 heads of 128 x 128: 409 us a call against 522 with the quads' walk;
// one prompt: 210 against 137.  Its 692 products a chunk and warp keep the tensor
// pipe 60 % busy in blocks of 64 columns.
#pragma once

#include "deltanet_chunk_parts.cuh"

namespace qfn {
namespace {

constexpr int kWarpCols = 128;
constexpr int kWarpStages = 3;
constexpr int kWarpThreads = kWarpCols / 16 * 32;

template <int DK>
struct WarpStage {
  unsigned char k[C * DK * 2], q[C * DK * 2];
  unsigned char t[3 * kTermBytes];
  float f[kFactors];
  unsigned char p[kPBytes];
  unsigned char v[C * kWarpCols * 2];
};

template <int DK>
struct WarpSmem {
  WarpStage<DK> stage[kWarpStages];
  uint64_t full[kWarpStages], empty[kWarpStages];
  int length[kSorted], seq;
};

// Values of a lane's columns g (first token bad0) and g + 8 (bad1) from those tokens on become NaN.
__device__ __forceinline__ void spoil(float (&d)[8][4], int bad0, int bad1) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int tok = i * 8 + 2 * (threadIdx.x & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (tok + (j & 1) >= (j < 2 ? bad0 : bad1)) d[i][j] = CUDART_NAN_F;
  }
}

// A warp walks 16 columns of S on its own, every product transposed so that the columns are the 16 rows
// of the A operand: the accumulators of one product, split into bf16 terms, are then the A fragments of
// the next, and S, R and d never leave the registers.  The k, q, T and P tiles are B operands that all
// warps of the block read from shared memory.
template <int DK>
__global__ void __launch_bounds__(kWarpThreads, 1) dn_walk_warp_kernel(const DnRows a, const Plan plan, const Work work,
                                                                       int64_t slot0, int64_t slot1, bool vec, int sms) {
  constexpr int kStages = kWarpStages, kVRow = kWarpCols * 2;
  extern __shared__ __align__(1024) unsigned char raw[];
  WarpSmem<DK>& sm = *reinterpret_cast<WarpSmem<DK>*>(raw);
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int cb = (a.dv + kWarpCols / 2 - 1) / (kWarpCols / 2);
  const int c0 = static_cast<int>(blockIdx.x % cb) * (kWarpCols / 2);
  const int h = static_cast<int>(blockIdx.x / cb % a.heads);
  pdl_wait();
  const Part part = choose(plan, blockIdx.x / cb / a.heads, slot0, slot1, sm.length, &sm.seq);
  if (part.none(slot1)) return;
  const int64_t seq = part.seq, begin = part.begin, len = part.len, base = part.base, first = part.first, last = part.last;
  const bool ok = part.ok;
  const int n = static_cast<int>(max(last - first, static_cast<int64_t>(0)));

  // Four warps have a scheduler each and walk a chunk of dk = 128 in 5.0 us, eight in 7.8.  Blocks have 128 columns, and
  // every second block of 64 none, but for sequences that would take longer so than their share of all SMs' time, where
  // these are few enough for all their blocks of 64 columns to run at once.
  bool wide = true;
  if (plan.n_seqs <= kSorted && ok) {
    const int64_t all = (slot1 - slot0) * a.heads * ((cb + 1) / 2);
    const int64_t sequences = plan.cu ? __syncthreads_count(tid < plan.n_seqs && (sm.length[tid] + C - 1) / C *
                                                                                    static_cast<int64_t>(sms) > all)
                                      : plan.n_seqs;
    wide = static_cast<int64_t>(n) * sms <= all || sequences * a.heads * cb > sms;
  }
  if (wide && (c0 & (kWarpCols / 2))) return;
  const int warps = min(wide ? kWarpCols / 16 : kWarpCols / 32, (a.dv - c0) / 16);   // those with columns
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 1 + warps * 32);   // the bulk copies' bytes, the lanes' copies of v
      mbar_init(&sm.empty[i], warps);
    }
    fence_mbar_init();
  }
  __syncthreads();

  if (w < warps) {
    constexpr int NT = DK / 8, KT = DK / 16;
    const float* s_from = first > 0 ? a.s_out : a.s_in;
    const int64_t s_at = (seq * a.heads + h) * DK * static_cast<int64_t>(a.dv) + c0 + w * 16 + g;
    float S[NT][4];   // S^T: rows are columns g and g + 8, columns are dk
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float* src = s_from + s_at + static_cast<int64_t>(i * 8 + 2 * t) * a.dv;
      S[i][0] = s_from ? src[0] : 0.f;
      S[i][1] = s_from ? src[a.dv] : 0.f;
      S[i][2] = s_from ? src[8] : 0.f;
      S[i][3] = s_from ? src[a.dv + 8] : 0.f;
      if (!ok) S[i][0] = S[i][1] = S[i][2] = S[i][3] = CUDART_NAN_F;
    }
    const int64_t pitch = static_cast<int64_t>(a.heads) * a.dv;
    // where this lane's pieces of a tile's fragments lie: rows of N, and rows of K (transposed)
    const int n_row = (lane & 7) + ((lane >> 4) << 3), n_ch = (lane >> 3) & 1, k_row = lane & 15, k_ch = lane >> 4;
    // Chunk `it` to its stage, this warp being done with the chunk before it there: its own columns of v; the
    // tiles that all warps read by the first, once all are done with it.
    auto copy = [&](int it) {
      const int st = it % kStages;
      WarpStage<DK>& sg = sm.stage[st];
      const int64_t t0 = begin + (first + it) * C, slot = base + first + it - slot0;
      const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
      const uint16_t* v = a.v + t0 * a.v_row + h * a.v_head + c0 + w * 16;
#pragma unroll
      for (int i = 0; i < C * 2 / 32; ++i) {
        const int r = i * 16 + (lane >> 1), ch = lane & 1;
        const uint32_t dst = smem_u32(sg.v) + swz<kVRow>(r, w * 2 + ch);
        const uint16_t* src = v + (r < cnt ? r * a.v_row + ch * 8 : 0);
        if (vec) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(r < cnt ? 16 : 0)
                       : "memory");
        } else {
          uint32_t u[4] = {0, 0, 0, 0};
          if (r < cnt)
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = src[2 * j] | static_cast<uint32_t>(src[2 * j + 1]) << 16;
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3])
                       : "memory");
        }
      }
      if (vec)
        asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(&sm.full[st])) : "memory");
      else
        mbar_arrive(&sm.full[st]);
      if (w == 0) {
        if (it >= kStages) wait(&sm.empty[st], (it / kStages + 1) & 1);
        if (lane == 0) {
          const int key_heads = a.heads / a.ratio;
          const unsigned char* head = work.heads + (slot * a.heads + h) * static_cast<int64_t>(kHeadBytes);
          mbar_arrive_expect_tx(&sm.full[st], 2 * C * DK * 2 + kHeadBytes);
          bulk_g2s(sg.k, work.kq + (slot * key_heads + h / a.ratio) * (2 * C * DK * 2), 2 * C * DK * 2, &sm.full[st]);
          bulk_g2s(sg.t, head, kHeadBytes, &sm.full[st]);
        }
        __syncwarp();
      }
    };
    asm volatile("fence.proxy.async.global;" ::: "memory");   // the other kernel's stores, before bulk copies of them
#pragma unroll 1
    for (int it = 0; it < n && it < kStages - 1; ++it) copy(it);
#pragma unroll 1
    for (int it = 0; it < n; ++it) {
      const int st = it % kStages;
      const WarpStage<DK>& sg = sm.stage[st];
      const uint32_t kb = smem_u32(sg.k), qb = smem_u32(sg.q);
      if (it + kStages - 1 < n) copy(it + kStages - 1);
      const float* f = sg.f;
      wait(&sm.full[st], (it / kStages) & 1);
      // S^T k and, from S's first two terms, S^T q: token tiles of 8
      float x[8][4], o[8][4];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        uint32_t s3[3][4];
        frag_split(S[2 * kt], S[2 * kt + 1], s3);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t y[4], z[4];
          const uint32_t at = swz<DK * 2>(b * 16 + n_row, kt * 2 + n_ch);
          ldsm4(y, kb + at);
          ldsm4(z, qb + at);
#pragma unroll
          for (int term = 0; term < 3; ++term)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (kt == 0 && term == 0) {
                mma_first(x[2 * b + j], s3[term], y[2 * j], y[2 * j + 1]);
                mma_first(o[2 * b + j], s3[term], z[2 * j], z[2 * j + 1]);
              } else {
                mma_add(x[2 * b + j], s3[term], y[2 * j], y[2 * j + 1]);
                if (term < 2) mma_add(o[2 * b + j], s3[term], z[2 * j], z[2 * j + 1]);
              }
            }
        }
      }
      // R = beta v - beta e^G S^T k
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t v[4];   // (columns 0-7 | 8-15) x (tokens 0-7), then tokens 8-15, transposed
        ldsm4t(v, smem_u32(sg.v) + swz<kVRow>(b * 16 + n_row, w * 2 + n_ch));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int i = 2 * b + j;
          const float2 fa = *reinterpret_cast<const float2*>(f + kFA + i * 8 + 2 * t);
          const float2 fb = *reinterpret_cast<const float2*>(f + kFB + i * 8 + 2 * t);
          x[i][0] = fmaf(fa.x, x[i][0], fb.x * __uint_as_float(v[2 * j] << 16));
          x[i][1] = fmaf(fa.y, x[i][1], fb.y * __uint_as_float(v[2 * j] & 0xffff0000u));
          x[i][2] = fmaf(fa.x, x[i][2], fb.x * __uint_as_float(v[2 * j + 1] << 16));
          x[i][3] = fmaf(fa.y, x[i][3], fb.y * __uint_as_float(v[2 * j + 1] & 0xffff0000u));
        }
      }
      // A token's infinity or NaN may not reach the tokens before it through T's and P's zeros: it is taken out
      // here and put back into d from that token on.
      int bad0 = C, bad1 = C;
      auto take_out = [&]() {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!(fabsf(x[i][j]) < CUDART_INF_F)) {
              (j < 2 ? bad0 : bad1) = min(j < 2 ? bad0 : bad1, i * 8 + 2 * t + (j & 1));
              x[i][j] = 0.f;
            }
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
          bad0 = min(bad0, __shfl_xor_sync(0xffffffffu, bad0, off));
          bad1 = min(bad1, __shfl_xor_sync(0xffffffffu, bad1, off));
        }
      };
      bool any_bad = any_not_finite(x);
      if (any_bad) take_out();
      // d = T R, blocks on and below the diagonal
      {
        float d[8][4];
        const uint32_t tb = smem_u32(sg.t) + lane * 16;
#pragma unroll
        for (int bj = 0; bj < 4; ++bj) {
          uint32_t r[3][4];
          frag_split(x[2 * bj], x[2 * bj + 1], r);
#pragma unroll
          for (int term = 2; term >= 0; --term) {   // of T, the smallest first; with it the terms of R that are not below 2^-24
            uint32_t y[4][4];
#pragma unroll
            for (int bi = bj; bi < 4; ++bi) ldsm4(y[bi], tb + term * kTermBytes + tri_block(bi, bj));
#pragma unroll
            for (int i = 2 - term; i >= 0; --i)
#pragma unroll
              for (int bi = bj; bi < 4; ++bi)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  if (bj == 0 && term == 2) mma_first(d[2 * bi + j], r[i], y[bi][2 * j], y[bi][2 * j + 1]);
                  else mma_add(d[2 * bi + j], r[i], y[bi][2 * j], y[bi][2 * j + 1]);
                }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i][j] = d[i][j];
      }
      if (any_bad) spoil(x, bad0, bad1);
      any_bad = any_not_finite(x);   // a d that overflowed is bad from its token on, too
      if (any_bad) take_out();
      // o = e^G S^T q + P d
      {
        const uint32_t pb = smem_u32(sg.p) + lane * 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 fq = *reinterpret_cast<const float2*>(f + kFQ + i * 8 + 2 * t);
          o[i][0] *= fq.x;
          o[i][1] *= fq.y;
          o[i][2] *= fq.x;
          o[i][3] *= fq.y;
        }
#pragma unroll
        for (int bj = 0; bj < 4; ++bj) {
          uint32_t d2[2][4];
          frag_split(x[2 * bj], x[2 * bj + 1], d2);
#pragma unroll
          for (int term = 1; term >= 0; --term) {   // of P
            uint32_t y[4][4];
#pragma unroll
            for (int bi = bj; bi < 4; ++bi) ldsm4(y[bi], pb + term * kTermBytes + tri_block(bi, bj));
#pragma unroll
            for (int i = 1 - term; i >= 0; --i)
#pragma unroll
              for (int bi = bj; bi < 4; ++bi)
#pragma unroll
                for (int j = 0; j < 2; ++j) mma_add(o[2 * bi + j], d2[i], y[bi][2 * j], y[bi][2 * j + 1]);
          }
        }
        if (any_bad) spoil(o, bad0, bad1);
        const int64_t t0 = begin + (first + it) * C;
        const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
        uint16_t* dst = a.out + (t0 + g) * pitch + static_cast<int64_t>(h) * a.dv + c0 + w * 16 + 2 * t;
#pragma unroll
        for (int i = 0; i < 8; ++i) {   // after the transposition a row is a token
          const __nv_bfloat162 b0 = __floats2bfloat162_rn(o[i][0], o[i][1]), b1 = __floats2bfloat162_rn(o[i][2], o[i][3]);
          const uint32_t y0 = transpose8x8(*reinterpret_cast<const uint32_t*>(&b0));
          const uint32_t y1 = transpose8x8(*reinterpret_cast<const uint32_t*>(&b1));
          if (i * 8 + g < cnt) {
            *reinterpret_cast<uint32_t*>(dst) = y0;
            *reinterpret_cast<uint32_t*>(dst + 8) = y1;
          }
          dst += 8 * pitch;
        }
      }
      // S = e^G64 S + d k
      if (any_bad) spoil(x, bad0, bad1);
      uint32_t wd[4][3][4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
#pragma unroll
        for (int i = 2 * b; i < 2 * b + 2; ++i) {
          const float2 fw = *reinterpret_cast<const float2*>(f + kFW + i * 8 + 2 * t);
          x[i][0] *= fw.x;
          x[i][1] *= fw.y;
          x[i][2] *= fw.x;
          x[i][3] *= fw.y;
        }
        frag_split(x[2 * b], x[2 * b + 1], wd[b]);
      }
      const float keep = f[kFEnd];
#pragma unroll
      for (int np = 0; np < NT / 4; ++np) {   // 32 of dk at a time
        float u[4][4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t y[4], z[4];
          ldsm4t(y, kb + swz<DK * 2>(b * 16 + k_row, np * 4 + k_ch));
          ldsm4t(z, kb + swz<DK * 2>(b * 16 + k_row, np * 4 + 2 + k_ch));
#pragma unroll
          for (int term = 0; term < 3; ++term) {
            if (b == 0 && term == 0) {
              mma_first(u[0], wd[b][term], y[0], y[1]);
              mma_first(u[1], wd[b][term], y[2], y[3]);
              mma_first(u[2], wd[b][term], z[0], z[1]);
              mma_first(u[3], wd[b][term], z[2], z[3]);
            } else {
              mma_add(u[0], wd[b][term], y[0], y[1]);
              mma_add(u[1], wd[b][term], y[2], y[3]);
              mma_add(u[2], wd[b][term], z[0], z[1]);
              mma_add(u[3], wd[b][term], z[2], z[3]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) S[np * 4 + i][j] = fmaf(S[np * 4 + i][j], keep, u[i][j]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[st]);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float* dst = a.s_out + s_at + static_cast<int64_t>(i * 8 + 2 * t) * a.dv;
      dst[0] = S[i][0];
      dst[a.dv] = S[i][1];
      dst[8] = S[i][2];
      dst[a.dv + 8] = S[i][3];
    }
    // nothing of this warp may still be on its way when the block ends
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
}

}  // namespace
}  // namespace qfn
