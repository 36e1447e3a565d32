// The gated delta rule over whole sequences (qfn_deltanet_chunk), 64 tokens at
// a time (the chunk form of qwen_engine.py:158-174's recurrence).
//
// With G_i the running sum of g in the chunk, k and q normalised, S the state
// before the chunk and j < i inside it:
//   A_ij = beta_i e^{G_i - G_j} (k_i . k_j)         T = (I + A)^-1
//   R_i  = beta_i (v_i - e^{G_i} S^T k_i)           d = T R
//   o_i  = e^{G_i} S^T q_i + sum_{j <= i} P_ij d_j  P_ij = e^{G_i - G_j} (q_i . k_j)
//   S'   = e^{G_64} S + sum_j e^{G_64 - G_j} k_j d_j^T
//
// Two kernels.  dn_prep_kernel does everything that does not need the state,
// a block per (chunk, key head): k and q as f16 rows, T, P and the decays of
// each token.  dn_chunk_kernel then walks a sequence's chunks, a block per
// (sequence, value head, 32 columns of S), with S in registers.
//
// Precision.  S leaves as fp32, so its factors need more than f16's 11 bits:
// every operand of an S or d product that is not exact is split into two f16
// terms (22 bits) after a power-of-two scale taken from its largest element;
// k and q rows are bf16 and exact in f16 after theirs.  The products that
// only reach the bf16 output (P d and S^T q) take one term.
#include "deltanet_batch.cuh"
#include "deltanet_chunk.cuh"

namespace qfn {
namespace {

constexpr int C = 64;            // tokens of a chunk
constexpr int kCols = 32;        // state columns of a block
constexpr int kStages = 3;       // chunks of what the recurrence reads
constexpr int kOutStages = 2;    // chunks of what only the outputs read
constexpr int kPrepThreads = 256;
constexpr int kThreads = 9 * 32; // 4 warps of the recurrence, 4 of the outputs, 1 of the copies
constexpr int kGS = 68;          // row pitch of the 64 x 64 fp32 matrices of dn_prep_kernel

// Per chunk and value head: T hi, T lo (f16, 128-byte rows, swizzled), the
// tokens' factors and the chunk's scales, then P (as T).
constexpr int kMat = C * C * 2;
enum { kFA = 0, kFB = C, kFQ = 2 * C, kFW = 3 * C, kFEnd = 4 * C };   // -beta e^G ck, beta, e^G cq, e^(G64 - G) ck
constexpr int kFactors = 4 * C + 4;   // + e^G64, scale of T, scale of P
constexpr int kRecBytes = 2 * kMat + kFactors * 4;
constexpr int kHeadBytes = kRecBytes + kMat;

__device__ unsigned int g_dn_status;

struct Work {
  unsigned char* kq;     // [slots][key heads][2][64][dk] f16
  unsigned char* heads;  // [slots][heads][kHeadBytes]
};

// Sequence n's tokens and its first chunk's slot.  Slots of neighbouring
// sequences never meet: cu / 64 rises by at least chunks - 1 per sequence.
struct Plan {
  const int32_t* cu;
  int64_t n_seqs, tokens;
  __device__ int64_t begin(int64_t n) const { return cu ? cu[n] : n * (tokens / n_seqs); }
  __device__ int64_t end(int64_t n) const { return cu ? cu[n + 1] : (n + 1) * (tokens / n_seqs); }
  __device__ int64_t slot(int64_t n) const { return begin(n) / C + n; }
};

__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }

// Exponent e with max * 2^e in [2^14, 2^15); any value of max gives 2^e and 2^-e as normal numbers.
__device__ __forceinline__ int scale_exp(uint32_t max_bits) {
  const int ex = static_cast<int>(max_bits >> 23) - 126;   // max in [2^(ex-1), 2^ex)
  return max_bits == 0 ? 0 : min(15 - ex, 120);
}

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b >= 0x7f800000u ? 0u : b;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two values as f16 hi and lo pairs (each scaled before).
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = pack_h2(a - f.x, b - f.y);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Byte offset of 16-byte piece `ch` of row `row` in a matrix of ROW-byte rows
// whose pieces are permuted so that eight rows' equal pieces lie in distinct banks.
template <int ROW>
__device__ __forceinline__ uint32_t swz(int row, int ch) {
  return static_cast<uint32_t>(row * ROW + ((ROW == 64 ? ch ^ ((row >> 1) & 3) : ch ^ (row & 7)) << 4));
}

// ------------------------------------------------------------------ what needs no state
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {   // kPrepThreads threads
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();   // red may still be read from the last call
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t m = red[0];
#pragma unroll
  for (int i = 1; i < kPrepThreads / 32; ++i) m = max(m, red[i]);
  return m;
}

template <int DK>
struct PrepSmem {
  union {
    struct {
      unsigned char k[C * DK * 2], q[C * DK * 2];   // f16 rows, swizzled
    };
    struct {
      float t[C * kGS];        // A, then T
      float y[3 * 16 * 20];    // a level's sums
    };
  };
  float gk[C * kGS], gq[C * kGS];   // k_i . k_j, q_i . k_j of the scaled rows
  double g[C];
  float ck[C], cq[C], beta[C];
  uint32_t red[kPrepThreads / 32];
};

// The inverse of I + A, A strictly lower triangular in t: 16 x 16 blocks on
// the diagonal by substitution, then T_ij = -T_ii sum_k A_ik T_kj diagonal by
// diagonal, in fp32.  Block T_ij below the diagonal is left at block (j, i),
// since A_ij is still needed: t_at gives an element's place.
__device__ __forceinline__ int t_at(int i, int j) { return ((j & ~15) + (i & 15)) * kGS + (i & ~15) + (j & 15); }

template <int DK>
__device__ __forceinline__ void invert(PrepSmem<DK>& sm) {
  const int tid = threadIdx.x;
  float x[16];
  const int b = tid >> 4, c = tid & 15;   // block, column (the first 64 threads)
  if (tid < 64) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) s = fmaf(-sm.t[(b * 16 + i) * kGS + b * 16 + j], x[j], s);
      x[i] = s;
    }
  }
  __syncthreads();
  if (tid < 64) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sm.t[(b * 16 + i) * kGS + b * 16 + c] = x[i];
  }
  // 64 threads per block of a diagonal: row r, columns c4 .. c4 + 3
  const int u = tid >> 6, r = (tid >> 2) & 15, c4 = (tid & 3) * 4;
#pragma unroll 1
  for (int d = 1; d < 4; ++d) {
    __syncthreads();
    const int bi = u + d, bj = u;
    const bool on = u < 4 - d;
    if (on) {
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = bj * 16; k < bi * 16; ++k) {
        const float a = sm.t[(bi * 16 + r) * kGS + k];
        const float4 w = *reinterpret_cast<const float4*>(&sm.t[t_at(k, bj * 16 + c4)]);
        y.x = fmaf(a, w.x, y.x); y.y = fmaf(a, w.y, y.y); y.z = fmaf(a, w.z, y.z); y.w = fmaf(a, w.w, y.w);
      }
      *reinterpret_cast<float4*>(&sm.y[u * 320 + r * 20 + c4]) = y;
    }
    __syncthreads();
    if (on) {
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float a = -sm.t[(bi * 16 + r) * kGS + bi * 16 + k];
        const float4 w = *reinterpret_cast<const float4*>(&sm.y[u * 320 + k * 20 + c4]);
        y.x = fmaf(a, w.x, y.x); y.y = fmaf(a, w.y, y.y); y.z = fmaf(a, w.z, y.z); y.w = fmaf(a, w.w, y.w);
      }
      *reinterpret_cast<float4*>(&sm.t[t_at(bi * 16 + r, bj * 16 + c4)]) = y;
    }
  }
  __syncthreads();
}

// One bf16 row of q or k (zero behind the sequence's end) as f16: the row's
// scale 2^e, its factor (1 / norm) 2^-e, the swizzled row in shared memory.
template <int DK>
__device__ __forceinline__ void f16_row(const float (&x)[DK / 32], unsigned char* tile, int row, float* factor,
                                        float divide) {
  const int lane = threadIdx.x & 31;
  float ss = 0.f;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < DK / 32; ++i) {
    ss = fmaf(x[i], x[i], ss);
    m = max(m, finite_bits(x[i]));
  }
  ss = warp_sum(ss);
  m = __reduce_max_sync(0xffffffffu, m);
  const int e = scale_exp(m);
  const float s = exp2i(e);
  // lane holds elements lane * (DK / 32) ...
  constexpr int kPer = DK / 32;
  const uint32_t at = swz<DK * 2>(row, lane * kPer / 8) + (lane * kPer % 8) * 2;
#pragma unroll
  for (int i = 0; i < kPer; i += 2)
    *reinterpret_cast<uint32_t*>(tile + at + i * 2) = pack_h2(x[i] * s, x[i + 1] * s);
  // a row of zeros counts for nothing: its factor, up to 1000, would take the others' digits.  (An
  // infinity has m = 0 too where nothing else is finite; its sum keeps it.)
  if (lane == 0) *factor = ss == 0.f ? 0.f : rsqrtf(ss + 1e-6f) / divide * exp2i(-e);
}

template <int DK>
__device__ __forceinline__ void load_row(const uint16_t* p, bool in, bool vec, float (&x)[DK / 32]) {
  const int lane = threadIdx.x & 31;
  constexpr int kPer = DK / 32;
  if (!in) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = 0.f;
    return;
  }
  p += lane * kPer;
  if (vec) {
#pragma unroll
    for (int i = 0; i < kPer; i += 2) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p + i);
      x[i] = __uint_as_float(w << 16);
      x[i + 1] = __uint_as_float(w & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = bf16_bits_to_f32(p[i]);
  }
}

template <int DK>
__global__ void __launch_bounds__(kPrepThreads) dn_prep_kernel(const DnRows a, const Plan plan, const Work work,
                                                               int64_t slot0, bool vec) {
  extern __shared__ __align__(1024) unsigned char raw[];
  PrepSmem<DK>& sm = *reinterpret_cast<PrepSmem<DK>*>(raw);
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int key_heads = a.heads / a.ratio;
  const int hk = static_cast<int>(blockIdx.x % key_heads);
  const int64_t slot = slot0 + blockIdx.x / key_heads;
  pdl_wait();
  pdl_launch_dependents();
  // the sequence whose slots hold this one: the last whose first slot is not past it
  int64_t n;
  if (plan.cu) {
    int count = 0;
    for (int64_t i = 0; i < plan.n_seqs; i += kPrepThreads)
      count += __syncthreads_count(i + tid < plan.n_seqs && plan.slot(i + tid) <= slot);
    n = count - 1;
    if (n < 0 || !dn_plan_ok(plan.cu, plan.n_seqs, plan.tokens)) return;
  } else {
    n = min(slot * C / (plan.tokens / plan.n_seqs + C) , plan.n_seqs - 1);
    while (n + 1 < plan.n_seqs && plan.slot(n + 1) <= slot) ++n;
  }
  const int64_t t0 = plan.begin(n) + (slot - plan.slot(n)) * C;
  const int cnt = static_cast<int>(min(static_cast<int64_t>(C), plan.end(n) - t0));
  if (cnt <= 0) return;

  // k and q rows: 8 of each per warp
  {
    const uint16_t* src[2] = {a.k + hk * a.k_head, a.q + hk * a.q_head};
    const int64_t row[2] = {a.k_row, a.q_row};
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float x[8][DK / 32];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = w * 8 + i;
        load_row<DK>(src[m] + (t0 + r) * row[m], r < cnt, vec, x[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        f16_row<DK>(x[i], m ? sm.q : sm.k, w * 8 + i, m ? &sm.cq[w * 8 + i] : &sm.ck[w * 8 + i], m ? a.q_scale : 1.f);
    }
  }
  __syncthreads();
  // the rows to the workspace, as they lie
  {
    uint4* dst = reinterpret_cast<uint4*>(work.kq + ((slot - slot0) * key_heads + hk) * (2 * C * DK * 2));
    const uint4* src = reinterpret_cast<const uint4*>(sm.k);
#pragma unroll
    for (int i = 0; i < 2 * C * DK * 2 / 16 / kPrepThreads; ++i) dst[i * kPrepThreads + tid] = src[i * kPrepThreads + tid];
  }
  // k_i . k_j (warps 0-3) and q_i . k_j (warps 4-7), 16 rows per warp, up to the diagonal's block
  {
    const int m = w & 3;
    const uint32_t rows = smem_u32(w < 4 ? sm.k : sm.q), cols = smem_u32(sm.k);
    float acc[8][4] = {};
#pragma unroll
    for (int kt = 0; kt < DK / 16; ++kt) {
      uint32_t x[4];
      ldsm4(x, rows + swz<DK * 2>(m * 16 + (lane & 15), kt * 2 + (lane >> 4)));
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        if (np > m) continue;
        uint32_t b[4];
        ldsm4(b, cols + swz<DK * 2>(np * 16 + (lane & 7) + ((lane >> 4) << 3), kt * 2 + ((lane >> 3) & 1)));
        mma_16816(acc[2 * np], x, b[0], b[1]);
        mma_16816(acc[2 * np + 1], x, b[2], b[3]);
      }
    }
    float* dst = w < 4 ? sm.gk : sm.gq;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j / 2 > m) continue;
      *reinterpret_cast<float2*>(&dst[(m * 16 + g) * kGS + j * 8 + 2 * t]) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(&dst[(m * 16 + g + 8) * kGS + j * 8 + 2 * t]) = make_float2(acc[j][2], acc[j][3]);
    }
  }
  __syncthreads();   // the k and q tiles are free for A and T from here

#pragma unroll 1
  for (int hv = 0; hv < a.ratio; ++hv) {
    const int h = hk * a.ratio + hv;
    unsigned char* dst = work.heads + ((slot - slot0) * a.heads + h) * static_cast<int64_t>(kHeadBytes);
    float* factors = reinterpret_cast<float*>(dst + 2 * kMat);
    // Running sum of g in 64 bits: differences of far tokens' sums keep their
    // digits.  exp(-200) is 0 in fp32, and a finite sum keeps exp(G_i - G_j) a number.
    if (w == 0) {
      double s[2];
      float bt[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        const float gv = r < cnt ? a.g[(t0 + r) * a.g_row + h * a.g_head] : 0.f;
        s[i] = gv < -200.f ? -200.f : gv;
        bt[i] = r < cnt ? bf16_bits_to_f32(a.beta[(t0 + r) * a.b_row + h * a.b_head]) : 0.f;
      }
      double run = s[0] + s[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      const double G[2] = {run - s[1], run};
      const double last = __shfl_sync(0xffffffffu, run, 31);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        sm.g[r] = G[i];
        sm.beta[r] = bt[i];
        const float eg = expf(static_cast<float>(G[i]));
        factors[kFA + r] = -bt[i] * eg * sm.ck[r];
        factors[kFB + r] = bt[i];
        factors[kFQ + r] = eg * sm.cq[r];
        factors[kFW + r] = expf(static_cast<float>(last - G[i])) * sm.ck[r];
      }
      if (lane == 0) factors[kFEnd] = expf(static_cast<float>(last));
    }
    __syncthreads();
    // A into t; P from registers
    float p[2][8];
    uint32_t pm = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int i = s * 32 + (tid >> 3), j0 = (tid & 7) * 8;
      const double gi = sm.g[i];
      const float bi = sm.beta[i] * sm.ck[i], qi = sm.cq[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int jj = j0 + j;
        float av = 0.f, pv = 0.f;
        if (jj <= i) {
          const float f = expf(static_cast<float>(gi - sm.g[jj])) * sm.ck[jj];
          pv = f * qi * sm.gq[i * kGS + jj];
          if (jj < i) av = f * bi * sm.gk[i * kGS + jj];
        }
        sm.t[i * kGS + jj] = av;
        p[s][j] = pv;
        pm = max(pm, finite_bits(pv));
      }
    }
    const int ep = scale_exp(block_max(pm, sm.red));
    {
      const float sc = exp2i(ep);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        *reinterpret_cast<uint4*>(dst + kRecBytes + swz<128>(s * 32 + (tid >> 3), tid & 7)) =
            make_uint4(pack_h2(p[s][0] * sc, p[s][1] * sc), pack_h2(p[s][2] * sc, p[s][3] * sc),
                       pack_h2(p[s][4] * sc, p[s][5] * sc), pack_h2(p[s][6] * sc, p[s][7] * sc));
    }
    invert(sm);
    uint32_t tm = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int i = s * 32 + (tid >> 3), j0 = (tid & 7) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[s][j] = j0 + j <= i ? sm.t[t_at(i, j0 + j)] : 0.f;
        tm = max(tm, finite_bits(p[s][j]));
      }
    }
    const int et = scale_exp(block_max(tm, sm.red));
    const float sc = exp2i(et);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) split2(p[s][2 * j] * sc, p[s][2 * j + 1] * sc, hi[j], lo[j]);
      const uint32_t at = swz<128>(s * 32 + (tid >> 3), tid & 7);
      *reinterpret_cast<uint4*>(dst + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(dst + kMat + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    if (tid == 0) {
      factors[kFEnd + 1] = exp2i(-et);
      factors[kFEnd + 2] = exp2i(-ep);
      factors[kFEnd + 3] = 0.f;
    }
    // the next head's A overwrites t only after the barriers before it
  }
}

// ------------------------------------------------------------------ the walk over the chunks
template <int DK>
struct Stage {
  unsigned char k[C * DK * 2];
  unsigned char t_hi[kMat], t_lo[kMat];
  float f[kFactors];
  unsigned char v[C * kCols * 2];
};
template <int DK>
struct OutStage {
  unsigned char q[C * DK * 2], p[kMat];
};

// Fragments travel as 16 bytes per lane.
template <int DK>
struct ChunkSmem {
  Stage<DK> stage[kStages];
  OutStage<DK> out_stage[kOutStages];
  uint4 s_hi[2][2][2][DK / 32][32];   // [buffer][columns][half of dk][k tile][lane]
  uint4 d_hi[2][2][2][2][32];         // [buffer][columns][half of the tokens][tile][lane]
  float4 x[2][2][4][32];              // partial S^T k [columns][half][..][lane]
  uint4 rx[2][2][2][2][32];           // R [columns][half][tile][hi, lo][lane]
  uint4 dx[2][2][2][2][32];           // weighted d, likewise
  int bad[2][2][16];                  // [buffer][columns][column] first token whose R is not finite, or C
  float s_inv[2][2][2], d_inv[2][2][2], r_inv[2][2], dx_inv[2][2];
  uint64_t full[kStages], empty[kStages], out_full[kOutStages], out_empty[kOutStages];
  uint64_t s_full[2][2], d_full[2][2], out_done[2][2];   // [buffer][columns]
};

// The wait is bounded; a failure is recorded and the walk goes on with what is there.
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity) {
  if (!mbar_wait(bar, parity)) atomicOr(&g_dn_status, kStatusTimeout);
  __syncwarp();
}

__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

__device__ __forceinline__ void pair_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, 64;" ::"r"(id + 1) : "memory");
}

// Largest finite magnitude of a warp's values as float bits.
template <int N>
__device__ __forceinline__ uint32_t warp_max(const float (&v)[N][4]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(v[i][j]));
  uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
  if (b >= 0x7f800000u) {   // an infinity somewhere: the other columns keep their own scale
    b = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) b = max(b, finite_bits(v[i][j]));
    b = __reduce_max_sync(0xffffffffu, b);
  }
  return b;
}

// Accumulators of two neighbouring 16 x 8 tiles as the hi and lo fragments of a 16 x 16 operand.
__device__ __forceinline__ void frag_split(const float (&a)[4], const float (&b)[4], float s, uint32_t (&hi)[4],
                                           uint32_t (&lo)[4]) {
  split2(a[0] * s, a[1] * s, hi[0], lo[0]);
  split2(a[2] * s, a[3] * s, hi[1], lo[1]);
  split2(b[0] * s, b[1] * s, hi[2], lo[2]);
  split2(b[2] * s, b[3] * s, hi[3], lo[3]);
}

__device__ __forceinline__ uint4 as_uint4(const uint32_t (&r)[4]) { return make_uint4(r[0], r[1], r[2], r[3]); }
__device__ __forceinline__ void from_uint4(uint32_t (&r)[4], uint4 v) { r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w; }

// Blocks of 16 tokens belong to the two warps of a pair so that their
// triangular products take the same time: 0 and 3 to one, 1 and 2 to the other.
__device__ __forceinline__ int block_of(int half, int i) { return half ? 1 + i : 3 * i; }

// The values of a lane's columns g (first token bad0) and g + 8 (bad1) from those tokens on become v.
__device__ __forceinline__ void spoil(float (&d)[4][4], int half, int bad0, int bad1, float v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int tok = block_of(half, i >> 1) * 16 + (i & 1) * 8 + 2 * (threadIdx.x & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (tok + (j & 1) >= (j < 2 ? bad0 : bad1)) d[i][j] = v;
  }
}

template <int DK>
__global__ void __launch_bounds__(kThreads, 1) dn_chunk_kernel(const DnRows a, const Plan plan, const Work work,
                                                               int64_t slot0, int64_t slot1, bool vec) {
  extern __shared__ __align__(1024) unsigned char raw[];
  ChunkSmem<DK>& sm = *reinterpret_cast<ChunkSmem<DK>*>(raw);
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int cb = a.dv / kCols;
  const int c0 = static_cast<int>(blockIdx.x % cb) * kCols;
  const int h = static_cast<int>(blockIdx.x / cb % a.heads);
  const int64_t seq = blockIdx.x / cb / a.heads;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 33);
      mbar_init(&sm.empty[i], 8);
    }
    for (int i = 0; i < kOutStages; ++i) {
      mbar_init(&sm.out_full[i], 1);
      mbar_init(&sm.out_empty[i], 4);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sm.s_full[0][0] + i, 2);
      mbar_init(&sm.d_full[0][0] + i, 2);
      mbar_init(&sm.out_done[0][0] + i, 2);
    }
    fence_mbar_init();
  }
  pdl_wait();
  const bool ok = !plan.cu || dn_plan_ok(plan.cu, plan.n_seqs, plan.tokens);
  __syncthreads();
  // this launch's chunks of the sequence
  const int64_t begin = ok ? plan.begin(seq) : 0, base = ok ? plan.slot(seq) : slot0;
  const int64_t len = ok ? plan.end(seq) - begin : 0, chunks = (len + C - 1) / C;
  const int64_t first = max(slot0 - base, static_cast<int64_t>(0)), last = min(slot1 - base, chunks);
  if (base >= slot1 || (first > 0 && first >= last)) return;
  const float* s_from = first > 0 ? a.s_out : a.s_in;
  const int64_t s_at = (seq * a.heads + h) * DK * static_cast<int64_t>(a.dv) + c0;

  if (w < 4) {
    // ---- the recurrence: columns grp * 16 .. + 15, a half of dk per warp
    constexpr int NT = DK / 16, KT = DK / 32;
    const int grp = w >> 1, half = w & 1, d0 = half * (DK / 2);
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
    for (int64_t ci = first; ci < last; ++ci) {
      const uint32_t it = static_cast<uint32_t>(ci - first), st = it % kStages, buf = it & 1;
      Stage<DK>& sg = sm.stage[st];
      // S as f16 terms; the hi terms also go to the warps of the outputs
      uint32_t hi[KT][4], lo[KT][4];
      float inv;
      {
        const int e = scale_exp(warp_max(S));
        const float s = exp2i(e);
        inv = exp2i(-e);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) frag_split(S[2 * kt], S[2 * kt + 1], s, hi[kt], lo[kt]);
      }
      if (it >= 2) wait(&sm.out_done[buf][grp], ((it >> 1) + 1) & 1);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) sm.s_hi[buf][grp][half][kt][lane] = as_uint4(hi[kt]);
      if (lane == 0) sm.s_inv[buf][grp][half] = inv;
      if (half == 0 && lane < 16) sm.bad[buf][grp][lane] = C;
      warp_arrive(&sm.s_full[buf][grp]);
      wait(&sm.full[st], (it / kStages) & 1);
      // this half's part of S^T k: token blocks in the order own, own, other, other
      const uint32_t kb = smem_u32(sg.k);
      float acc[8][4] = {};
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int blk = block_of(b < 2 ? half : half ^ 1, b & 1);
          uint32_t x[4];
          ldsm4(x, kb + swz<DK * 2>(blk * 16 + (lane & 7) + ((lane >> 4) << 3), d0 / 8 + kt * 2 + ((lane >> 3) & 1)));
          mma_16816(acc[2 * b], hi[kt], x[0], x[1]);
          mma_16816(acc[2 * b + 1], hi[kt], x[2], x[3]);
          mma_16816(acc[2 * b], lo[kt], x[0], x[1]);
          mma_16816(acc[2 * b + 1], lo[kt], x[2], x[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sm.x[grp][half][i][lane] =
            make_float4(acc[4 + i][0] * inv, acc[4 + i][1] * inv, acc[4 + i][2] * inv, acc[4 + i][3] * inv);
      pair_sync(grp);
      // R of the own blocks
      float R[4][4];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int tb = block_of(half, b) * 16;
        uint32_t v[4];   // (columns 0-7 | 8-15) x (tokens 0-7), then tokens 8-15, transposed
        ldsm4t(v, smem_u32(sg.v) + swz<64>(tb + (lane & 7) + ((lane >> 4) << 3), grp * 2 + ((lane >> 3) & 1)));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 o = sm.x[grp][half ^ 1][2 * b + j][lane];
          const float2 fa = *reinterpret_cast<const float2*>(&sg.f[kFA + tb + j * 8 + 2 * t]);
          const float2 fb = *reinterpret_cast<const float2*>(&sg.f[kFB + tb + j * 8 + 2 * t]);
          const int i = 2 * b + j;
          const uint32_t v0 = v[2 * j], v1 = v[2 * j + 1];
          R[i][0] = fmaf(fa.x, fmaf(acc[i][0], inv, o.x), fb.x * __uint_as_float(v0 << 16));
          R[i][1] = fmaf(fa.y, fmaf(acc[i][1], inv, o.y), fb.y * __uint_as_float(v0 & 0xffff0000u));
          R[i][2] = fmaf(fa.x, fmaf(acc[i][2], inv, o.z), fb.x * __uint_as_float(v1 << 16));
          R[i][3] = fmaf(fa.y, fmaf(acc[i][3], inv, o.w), fb.y * __uint_as_float(v1 & 0xffff0000u));
        }
      }
      uint32_t rh[2][4], rl[2][4];
      float r_inv;
      {
        // A token's infinity or NaN may not reach the tokens before it through T's and P's zeros:
        // it is taken out here and put back into d from that token on.
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(R[i][j]) & 0x7fffffffu);
        m = __reduce_max_sync(0xffffffffu, m);
        if (m >= 0x7f800000u) {
          m = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if ((__float_as_uint(R[i][j]) & 0x7fffffffu) >= 0x7f800000u) {
                atomicMin(&sm.bad[buf][grp][g + (j >> 1) * 8], block_of(half, i >> 1) * 16 + (i & 1) * 8 + 2 * t + (j & 1));
                R[i][j] = 0.f;
              }
              m = max(m, __float_as_uint(R[i][j]) & 0x7fffffffu);
            }
          m = __reduce_max_sync(0xffffffffu, m);
        }
        const int e = scale_exp(m);
        const float s = exp2i(e);
        r_inv = exp2i(-e);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          frag_split(R[2 * b], R[2 * b + 1], s, rh[b], rl[b]);
          sm.rx[grp][half][b][0][lane] = as_uint4(rh[b]);
          sm.rx[grp][half][b][1][lane] = as_uint4(rl[b]);
        }
        if (lane == 0) sm.r_inv[grp][half] = r_inv;
      }
      pair_sync(grp);
      // d = T R of the own blocks
      float own[4][4] = {}, oth[4][4] = {};
      const uint32_t th = smem_u32(sg.t_hi), tl = smem_u32(sg.t_lo);
#pragma unroll
      for (int s = 0; s < 4; ++s) {   // source block: own, own, other, other
        const int bj = block_of(s < 2 ? half : half ^ 1, s & 1);
        uint32_t xh[4], xl[4];
        if (s < 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) { xh[i] = rh[s & 1][i]; xl[i] = rl[s & 1][i]; }
        } else {
          from_uint4(xh, sm.rx[grp][half ^ 1][s & 1][0][lane]);
          from_uint4(xl, sm.rx[grp][half ^ 1][s & 1][1][lane]);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int bi = block_of(half, b);
          if (bj > bi) continue;
          uint32_t yh[4], yl[4];
          const uint32_t at = swz<128>(bi * 16 + (lane & 7) + ((lane >> 4) << 3), bj * 2 + ((lane >> 3) & 1));
          ldsm4(yh, th + at);
          ldsm4(yl, tl + at);
          float(*d)[4] = s < 2 ? own : oth;
          mma_16816(d[2 * b], xh, yh[0], yh[1]);
          mma_16816(d[2 * b + 1], xh, yh[2], yh[3]);
          mma_16816(d[2 * b], xl, yh[0], yh[1]);
          mma_16816(d[2 * b + 1], xl, yh[2], yh[3]);
          mma_16816(d[2 * b], xh, yl[0], yl[1]);
          mma_16816(d[2 * b + 1], xh, yl[2], yl[3]);
        }
      }
      {
        const float t_inv = sg.f[kFEnd + 1];
        const float so = r_inv * t_inv, sx = sm.r_inv[grp][half ^ 1] * t_inv;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) own[i][j] = fmaf(oth[i][j], sx, own[i][j] * so);
      }
      const int bad0 = sm.bad[buf][grp][g], bad1 = sm.bad[buf][grp][g + 8];
      const bool any_bad = __any_sync(0xffffffffu, bad0 < C || bad1 < C);
      if (any_bad) spoil(own, half, bad0, bad1, 0.f);
      // d in f16 for the outputs, weighted and in two terms for the state
      {
        const int e = scale_exp(warp_max(own));
        const float s = exp2i(e);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float(&p)[4] = own[2 * b];
          const float(&q)[4] = own[2 * b + 1];
          sm.d_hi[buf][grp][half][b][lane] = make_uint4(pack_h2(p[0] * s, p[1] * s), pack_h2(p[2] * s, p[3] * s),
                                                        pack_h2(q[0] * s, q[1] * s), pack_h2(q[2] * s, q[3] * s));
        }
        if (lane == 0) sm.d_inv[buf][grp][half] = exp2i(-e);
      }
      warp_arrive(&sm.d_full[buf][grp]);
      if (any_bad) spoil(own, half, bad0, bad1, CUDART_NAN_F);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 fw = *reinterpret_cast<const float2*>(&sg.f[kFW + block_of(half, b) * 16 + j * 8 + 2 * t]);
          own[2 * b + j][0] *= fw.x;
          own[2 * b + j][1] *= fw.y;
          own[2 * b + j][2] *= fw.x;
          own[2 * b + j][3] *= fw.y;
        }
      float d_inv;
      {
        const int e = scale_exp(warp_max(own));
        const float s = exp2i(e);
        d_inv = exp2i(-e);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          frag_split(own[2 * b], own[2 * b + 1], s, rh[b], rl[b]);
          sm.dx[grp][half][b][0][lane] = as_uint4(rh[b]);
          sm.dx[grp][half][b][1][lane] = as_uint4(rl[b]);
        }
        if (lane == 0) sm.dx_inv[grp][half] = d_inv;
      }
      pair_sync(grp);
      // S = e^G64 S + d k^T for this half of dk
      const float eg = sg.f[kFEnd];
#pragma unroll
      for (int s = 0; s < 2; ++s) {   // the own tokens, then the other warp's
        float u[NT][4] = {};
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int blk = block_of(s ? half ^ 1 : half, b);
          uint32_t xh[4], xl[4];
          if (s == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { xh[i] = rh[b][i]; xl[i] = rl[b][i]; }
          } else {
            from_uint4(xh, sm.dx[grp][half ^ 1][b][0][lane]);
            from_uint4(xl, sm.dx[grp][half ^ 1][b][1][lane]);
          }
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            uint32_t y[4];
            ldsm4t(y, kb + swz<DK * 2>(blk * 16 + (lane & 15), d0 / 8 + np * 2 + (lane >> 4)));
            mma_16816(u[2 * np], xh, y[0], y[1]);
            mma_16816(u[2 * np + 1], xh, y[2], y[3]);
            mma_16816(u[2 * np], xl, y[0], y[1]);
            mma_16816(u[2 * np + 1], xl, y[2], y[3]);
          }
        }
        const float us = s ? sm.dx_inv[grp][half ^ 1] : d_inv;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) S[i][j] = fmaf(u[i][j], us, s ? S[i][j] : S[i][j] * eg);
      }
      warp_arrive(&sm.empty[st]);
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
  } else if (w < 8) {
    // ---- the outputs: columns grp * 16 .. + 15, half of the token blocks per warp
    constexpr int KT = DK / 32;
    const int grp = (w - 4) >> 1, half = w & 1;
    for (int64_t ci = first; ci < last; ++ci) {
      const uint32_t it = static_cast<uint32_t>(ci - first), st = it % kStages, so = it % kOutStages, buf = it & 1;
      Stage<DK>& sg = sm.stage[st];
      OutStage<DK>& og = sm.out_stage[so];
      const int64_t t0 = begin + ci * C;
      const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
      float o[4][4];
      wait(&sm.full[st], (it / kStages) & 1);
      wait(&sm.out_full[so], (it / kOutStages) & 1);
      wait(&sm.s_full[buf][grp], (it >> 1) & 1);
      const uint32_t qb = smem_u32(og.q), pb = smem_u32(og.p);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {   // halves of dk: each has its own scale
        float acc[4][4] = {};
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          uint32_t x[4];
          from_uint4(x, sm.s_hi[buf][grp][hf][kt][lane]);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            uint32_t y[4];
            ldsm4(y, qb + swz<DK * 2>(block_of(half, b) * 16 + (lane & 7) + ((lane >> 4) << 3),
                                      hf * (DK / 16) + kt * 2 + ((lane >> 3) & 1)));
            mma_16816(acc[2 * b], x, y[0], y[1]);
            mma_16816(acc[2 * b + 1], x, y[2], y[3]);
          }
        }
        const float s = sm.s_inv[buf][grp][hf];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][j] = hf ? fmaf(acc[i][j], s, o[i][j]) : acc[i][j] * s;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = *reinterpret_cast<const float2*>(&sg.f[kFQ + block_of(half, i >> 1) * 16 + (i & 1) * 8 + 2 * t]);
        o[i][0] *= f.x; o[i][1] *= f.y; o[i][2] *= f.x; o[i][3] *= f.y;
      }
      wait(&sm.d_full[buf][grp], (it >> 1) & 1);
      const float p_inv = sg.f[kFEnd + 2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {   // the tokens of either warp of the recurrence
        float acc[4][4] = {};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int bj = block_of(hf, s);
          uint32_t x[4];
          from_uint4(x, sm.d_hi[buf][grp][hf][s][lane]);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int bi = block_of(half, b);
            if (bj > bi) continue;
            uint32_t y[4];
            ldsm4(y, pb + swz<128>(bi * 16 + (lane & 7) + ((lane >> 4) << 3), bj * 2 + ((lane >> 3) & 1)));
            mma_16816(acc[2 * b], x, y[0], y[1]);
            mma_16816(acc[2 * b + 1], x, y[2], y[3]);
          }
        }
        const float s = sm.d_inv[buf][grp][hf] * p_inv;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][j] = fmaf(acc[i][j], s, o[i][j]);
      }
      {
        const int bad0 = sm.bad[buf][grp][g], bad1 = sm.bad[buf][grp][g + 8];
        if (__any_sync(0xffffffffu, bad0 < C || bad1 < C)) spoil(o, half, bad0, bad1, CUDART_NAN_F);
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
    }
  } else {
    // ---- the copies
    asm volatile("fence.proxy.async.global;" ::: "memory");   // the other kernel's stores, before bulk copies of them
    const int key_heads = a.heads / a.ratio;
    for (int64_t ci = first; ci < last; ++ci) {
      const uint32_t it = static_cast<uint32_t>(ci - first), st = it % kStages, so = it % kOutStages;
      Stage<DK>& sg = sm.stage[st];
      OutStage<DK>& og = sm.out_stage[so];
      const int64_t t0 = begin + ci * C, slot = base + ci - slot0;
      const unsigned char* kq = work.kq + (slot * key_heads + h / a.ratio) * (2 * C * DK * 2);
      const unsigned char* head = work.heads + (slot * a.heads + h) * static_cast<int64_t>(kHeadBytes);
      const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
      if (it >= kStages) wait(&sm.empty[st], (it / kStages + 1) & 1);
      if (lane == 0) {
        mbar_arrive_expect_tx(&sm.full[st], C * DK * 2 + kRecBytes);
        bulk_g2s(sg.k, kq, C * DK * 2, &sm.full[st]);
        bulk_g2s(sg.t_hi, head, kRecBytes, &sm.full[st]);
      }
      __syncwarp();
      const uint16_t* v = a.v + t0 * a.v_row + h * a.v_head + c0;
#pragma unroll
      for (int i = 0; i < C * kCols * 2 / 16 / 32; ++i) {
        const int r = i * 8 + (lane >> 2), ch = lane & 3;
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
        asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(&sm.full[st])) : "memory");
      else
        mbar_arrive(&sm.full[st]);
      if (it >= kOutStages) wait(&sm.out_empty[so], (it / kOutStages + 1) & 1);
      if (lane == 0) {
        mbar_arrive_expect_tx(&sm.out_full[so], C * DK * 2 + kMat);
        bulk_g2s(og.q, kq + C * DK * 2, C * DK * 2, &sm.out_full[so]);
        bulk_g2s(og.p, head + kRecBytes, kMat, &sm.out_full[so]);
      }
      __syncwarp();
    }
    // nothing of this warp may still be on its way when the block ends
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
}

}  // namespace

// ------------------------------------------------------------------ host
namespace {

// Chunks are taken in segments whose workspace stays within this, so that
// what dn_prep_kernel writes is still in L2 when dn_chunk_kernel reads it.
constexpr int64_t kSegmentBytes = int64_t{128} << 20;

int64_t slot_bytes(int n_heads, int n_key_heads, int dk) {
  return static_cast<int64_t>(n_key_heads) * 2 * C * dk * 2 + static_cast<int64_t>(n_heads) * kHeadBytes;
}
int64_t segment_slots(int64_t slots, int n_heads, int n_key_heads, int dk) {
  const int64_t fit = kSegmentBytes / slot_bytes(n_heads, n_key_heads, dk);
  return slots < fit ? slots : fit > 1 ? fit : 1;
}

template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, int64_t blocks, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int DK>
int run(const DnRows& a, const int32_t* cu, int64_t n_seqs, int64_t tokens, void* workspace, qfn_stream_t stream) {
  constexpr const char* what = "qfn_deltanet_chunk";
  const int key_heads = a.heads / a.ratio;
  const int64_t slots = tokens / C + n_seqs, seg = segment_slots(slots, a.heads, key_heads, DK);
  const int64_t blocks = n_seqs * a.heads * (a.dv / kCols);
  QFN_REQUIRE(blocks <= 0x7fffffff && seg * key_heads <= 0x7fffffff, QFN_ERR_UNSUPPORTED, "%s: too many sequences",
              what);
  auto even = [](const void* p, int64_t row, int64_t head, int64_t elems) {
    return aligned(p, 2 * elems) && row % elems == 0 && head % elems == 0;
  };
  const bool kq_vec = even(a.q, a.q_row, a.q_head, 2) && even(a.k, a.k_row, a.k_head, 2);
  const bool v_vec = even(a.v, a.v_row, a.v_head, 8);
  cudaError_t e = cudaFuncSetAttribute(dn_prep_kernel<DK>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       sizeof(PrepSmem<DK>));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(dn_chunk_kernel<DK>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(ChunkSmem<DK>));
  if (e != cudaSuccess) return set_error(QFN_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
  const Plan plan{cu, n_seqs, tokens};
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const Work work{ws, ws + seg * key_heads * (2 * C * DK * 2)};
  for (int64_t s0 = 0; s0 < slots && e == cudaSuccess; s0 += seg) {
    const int64_t s1 = s0 + seg < slots ? s0 + seg : slots;
    e = launch(dn_prep_kernel<DK>, (s1 - s0) * key_heads, kPrepThreads, sizeof(PrepSmem<DK>), as_stream(stream), a, plan,
               work, s0, kq_vec);
    if (e == cudaSuccess)
      e = launch(dn_chunk_kernel<DK>, blocks, kThreads, sizeof(ChunkSmem<DK>), as_stream(stream), a, plan, work, s0, s1,
                 v_vec);
  }
  if (e != cudaSuccess) return set_error(QFN_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace

bool dn_chunk_takes(int64_t tokens, int dk) { return dk <= 128 && tokens > kRecurrenceTokens; }

size_t dn_chunk_workspace(int64_t tokens, int64_t n_seqs, int n_heads, int n_key_heads, int dk) {
  const int64_t slots = tokens / C + n_seqs;
  return static_cast<size_t>(segment_slots(slots, n_heads, n_key_heads, dk) * slot_bytes(n_heads, n_key_heads, dk));
}

int dn_chunk(const DnRows& a, const int32_t* cu, int64_t n_seqs, int64_t tokens, int dk, void* workspace,
             qfn_stream_t stream) {
  return dk == 64 ? run<64>(a, cu, n_seqs, tokens, workspace, stream)
                  : run<128>(a, cu, n_seqs, tokens, workspace, stream);
}

int dn_chunk_status(unsigned int* v, bool clear) {
  unsigned int s = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&s, g_dn_status, sizeof(s));
  const unsigned int zero = 0;
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(g_dn_status, &zero, sizeof(zero));
  if (e != cudaSuccess) return set_error(QFN_ERR_CUDA, "deltanet status: %s", cudaGetErrorString(e));
  *v = s;
  return QFN_OK;
}

}  // namespace qfn
