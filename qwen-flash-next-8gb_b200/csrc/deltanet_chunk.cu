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
// a block per (chunk, key head): k and q as rows, T, P and the decays of each
// token.  A walk over a sequence's chunks follows, with S in registers:
// dn_walk_quad_kernel for few sequences, dn_walk_warp_kernel for many.
//
// Precision.  S, d and R are fp32 sums, and the tensor cores take them, and T,
// as three bf16 terms (24 bits, fp32's range): products of a three-term operand
// with k are exact, T R leaves out what is below 2^-24 of its terms.  k and q rows
// are bf16 as they come; their norms' reciprocals are in the tokens' factors.  The
// products that only reach the bf16 output, P d and S^T q, take two terms of P, d
// and S: 2^-16 before a rounding to 2^-9.
// (Before, one power-of-two scale and two f16 terms served 16 columns and 64
// tokens: values 2^-20 of the largest there lost their digits.)
//
// What bounds it: not the bytes (2048 tokens of 32 heads of 128 x 128 take 137 us,
// their bytes 10.6) but the preparation's latency and instructions (45 us on its
// own: 17,000 warp instructions a block, 41 % of the issue slots) and the walk's
// chain of chunks.  Chunks of 64 keep that chain short and T invertible in one block; token
// by token the same call takes 3.6 ms.
#include <atomic>

#include "deltanet_chunk.cuh"
#include "deltanet_chunk_parts.cuh"
#include "deltanet_walk_quad.cuh"
#include "deltanet_walk_warp.cuh"

namespace qfn {
namespace {

// ------------------------------------------------------------------ what needs no state
template <int DK>
struct PrepSmem {
  union {
    struct {
      unsigned char k[C * DK * 2], q[C * DK * 2];   // bf16 rows, swizzled
    };
    struct {
      float t[C * kGS];     // A, then T
      float y[32 * 36];     // A21 T11
    };
  };
  float gk[C * kGS], gq[C * kGS];   // k_i . k_j, q_i . k_j of the rows as they are
  float g_hi[C], g_lo[C], ck[C], cq[C], beta[C];
};

// Four neighbouring sums over k < N of row[k] m[k][0 .. 3], in fp32.  LOWER: only k <= r, the part of a lower
// triangular row r that is not zero (zeros would let a NaN of a later row into this one).
template <int N, bool LOWER>
__device__ __forceinline__ float4 row_product(const float* row, const float* m, int pitch, int r) {
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < N; k += 4) {
    const float4 av = *reinterpret_cast<const float4*>(row + k);
    const float ak[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 b = *reinterpret_cast<const float4*>(m + (k + i) * pitch);
      if (!LOWER || k + i <= r) {
        y.x = fmaf(ak[i], b.x, y.x); y.y = fmaf(ak[i], b.y, y.y); y.z = fmaf(ak[i], b.z, y.z); y.w = fmaf(ak[i], b.w, y.w);
      }
    }
  }
  return y;
}

// The inverse of I + A, A strictly lower triangular in t, in fp32: the four 16 x 16 blocks of the diagonal by
// substitution, a column per lane, then T21 = -T22 (A21 T11) twice, for the two 32 x 32 halves and for the whole.
// 4,400 cycles where the block has an SM to itself; two blocks of 32 and one merge take 7,200.
template <int DK>
__device__ __forceinline__ void invert(PrepSmem<DK>& sm) {
  const int tid = threadIdx.x;
  if (tid < 64) {
    const int c = tid & 15;
    float* t = sm.t + (tid >> 4) * 16 * (kGS + 1);
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s[4] = {i == c ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < i; j += 4) {
        const float4 r = *reinterpret_cast<const float4*>(t + i * kGS + j);   // zero from the diagonal on
        s[0] = fmaf(-r.x, x[j], s[0]);
        if (j + 1 < i) s[1] = fmaf(-r.y, x[j + 1], s[1]);
        if (j + 2 < i) s[2] = fmaf(-r.z, x[j + 2], s[2]);
        if (j + 3 < i) s[3] = fmaf(-r.w, x[j + 3], s[3]);
      }
      x[i] = (s[0] + s[1]) + (s[2] + s[3]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i * kGS + c] = x[i];
  }
  __syncthreads();
  {   // half p: a thread of the first 128 has row r, columns c4 .. c4 + 3
    const int p = (tid >> 6) & 1, r = (tid >> 2) & 15, c4 = (tid & 3) * 4;
    float* t = sm.t + p * 32 * (kGS + 1);
    float* y = sm.y + p * 16 * 20;
    if (tid < 128) *reinterpret_cast<float4*>(&y[r * 20 + c4]) = row_product<16, false>(t + (16 + r) * kGS, t + c4, kGS, r);
    __syncthreads();
    if (tid < 128) {
      const float4 v = row_product<16, true>(t + (16 + r) * kGS + 16, y + c4, 20, r);
      *reinterpret_cast<float4*>(&t[(16 + r) * kGS + c4]) = make_float4(-v.x, -v.y, -v.z, -v.w);
    }
    __syncthreads();
  }
  const int r = tid >> 3, c4 = (tid & 7) * 4;
  *reinterpret_cast<float4*>(&sm.y[r * 36 + c4]) = row_product<32, false>(sm.t + (32 + r) * kGS, sm.t + c4, kGS, r);
  __syncthreads();
  const float4 v = row_product<32, true>(sm.t + (32 + r) * kGS + 32, sm.y + c4, 36, r);
  *reinterpret_cast<float4*>(&sm.t[(32 + r) * kGS + c4]) = make_float4(-v.x, -v.y, -v.z, -v.w);
  __syncthreads();
}

// DK / 8 bf16 of a row, 16 bytes at a time.
template <int DK>
__device__ __forceinline__ void load_row(const uint16_t* p, bool in, bool vec, uint4 (&x)[DK / 64]) {
#pragma unroll
  for (int i = 0; i < DK / 64; ++i) {
    x[i] = make_uint4(0, 0, 0, 0);
    if (!in) continue;
    if (vec) {
      x[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      uint32_t u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = p[i * 8 + 2 * j] | static_cast<uint32_t>(p[i * 8 + 2 * j + 1]) << 16;
      x[i] = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
}

// Eight lanes hold a bf16 row of q or k: to shared memory and to the workspace, both swizzled; the row's factor.
template <int DK>
__device__ __forceinline__ void keep_row(const uint4 (&x)[DK / 64], unsigned char* tile, unsigned char* copy, int row,
                                         float* factor, float divide) {
  const int part = threadIdx.x & 7;
  float ss[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < DK / 64; ++i) {
    const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float lo = __uint_as_float(u[j] << 16), hi = __uint_as_float(u[j] & 0xffff0000u);
      ss[0] = fmaf(lo, lo, ss[0]);
      ss[1] = fmaf(hi, hi, ss[1]);
    }
    const uint32_t at = swz<DK * 2>(row, part * (DK / 64) + i);
    *reinterpret_cast<uint4*>(tile + at) = x[i];
    *reinterpret_cast<uint4*>(copy + at) = x[i];
  }
  float s = ss[0] + ss[1];
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (part == 0) *factor = rsqrtf(s + 1e-6f) / divide;
}

// Eight neighbouring values of a row as N terms, a matrix apart.
template <int N>
__device__ __forceinline__ void store_terms(const float (&v)[8], unsigned char* dst) {
  uint32_t u[4][N];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(v[2 * i], v[2 * i + 1], u[i]);
#pragma unroll
  for (int n = 0; n < N; ++n)
    *reinterpret_cast<uint4*>(dst + n * kTermBytes) = make_uint4(u[0][n], u[1][n], u[2][n], u[3][n]);
}

template <int DK>
__global__ void __launch_bounds__(kPrepThreads, 3) dn_prep_kernel(const DnRows a, const Plan plan, const Work work,
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
    n = plan.n_seqs == 1 ? 0 : min(slot * C / (plan.each + C), plan.n_seqs - 1);
    while (n + 1 < plan.n_seqs && plan.slot(n + 1) <= slot) ++n;
  }
  const int64_t t0 = plan.begin(n) + (slot - plan.slot(n)) * C;
  const int cnt = static_cast<int>(min(static_cast<int64_t>(C), plan.end(n) - t0));
  if (cnt <= 0) return;

  // g and beta of tokens 2 lane and 2 lane + 1 for warp 0's running sum, a head ahead of it
  float gv[2] = {0.f, 0.f};
  uint16_t bv[2] = {0, 0};
  auto request = [&](int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 2 * lane + i;
      if (w == 0 && r < cnt) {
        gv[i] = a.g[(t0 + r) * a.g_row + h * a.g_head];
        bv[i] = a.beta[(t0 + r) * a.b_row + h * a.b_head];
      }
    }
  };
  request(hk * a.ratio);
  // k and q rows: a warp takes four rows at a time, eight of each in all
  {
    const uint16_t* src[2] = {a.k + hk * a.k_head + (lane & 7) * (DK / 8), a.q + hk * a.q_head + (lane & 7) * (DK / 8)};
    const int64_t pitch[2] = {a.k_row, a.q_row};
    unsigned char* copy = work.kq + ((slot - slot0) * key_heads + hk) * (2 * C * DK * 2);
    uint4 x[4][DK / 64];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = w * 8 + (i & 1) * 4 + (lane >> 3);
      load_row<DK>(src[i >> 1] + (t0 + r) * pitch[i >> 1], r < cnt, vec, x[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = w * 8 + (i & 1) * 4 + (lane >> 3);
      keep_row<DK>(x[i], i < 2 ? sm.k : sm.q, copy + (i < 2 ? 0 : C * DK * 2), r, i < 2 ? &sm.ck[r] : &sm.cq[r],
                   i < 2 ? 1.f : a.q_scale);
    }
  }
  __syncthreads();
  // k_i . k_j (warps 0-3) and q_i . k_j (warps 4-7), 16 rows per warp, up to the diagonal's block
  {
    const int m = w & 3, g = lane >> 2, t = lane & 3;
    const uint32_t rows = smem_u32(w < 4 ? sm.k : sm.q), cols = smem_u32(sm.k);
    float acc[8][4] = {};
#pragma unroll 2
    for (int kt = 0; kt < DK / 16; ++kt) {
      uint32_t x[4];
      ldsm4(x, rows + swz<DK * 2>(m * 16 + (lane & 15), kt * 2 + (lane >> 4)));
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        if (np > m) continue;
        uint32_t b[4];
        ldsm4(b, cols + swz<DK * 2>(np * 16 + (lane & 7) + ((lane >> 4) << 3), kt * 2 + ((lane >> 3) & 1)));
        mma_add(acc[2 * np], x, b[0], b[1]);
        mma_add(acc[2 * np + 1], x, b[2], b[3]);
      }
    }
    float* dst = w < 4 ? sm.gk : sm.gq;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j / 2 > m) continue;
      *reinterpret_cast<float2*>(&dst[(m * 16 + g) * kGS + j * 8 + 2 * t]) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(&dst[(m * 16 + g + 8) * kGS + j * 8 + 2 * t]) = make_float2(acc[j][2], acc[j][3]);
    }
  }
  // the k and q tiles are free for A and T after the barrier below

#pragma unroll 1
  for (int hv = 0; hv < a.ratio; ++hv) {
    const int h = hk * a.ratio + hv;
    unsigned char* dst = work.heads + ((slot - slot0) * a.heads + h) * static_cast<int64_t>(kHeadBytes);
    float* factors = reinterpret_cast<float*>(dst + 3 * kTermBytes);
    // Running sum of g in 64 bits, kept as two floats: differences of far tokens' sums keep their
    // digits.  exp(-200) is 0 in fp32, and a finite sum keeps exp(G_i - G_j) a number.
    if (w == 0) {
      double s[2];
      float bt[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = gv[i] < -200.f ? -200.f : gv[i];
        bt[i] = bf16_bits_to_f32(bv[i]);
      }
      if (hv + 1 < a.ratio) request(h + 1);
      double run = s[0] + s[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      const double before = __shfl_up_sync(0xffffffffu, run, 1);   // not run - s[1]: s[1] may be NaN
      const double G[2] = {lane ? before + s[0] : s[0], run};
      const double last = __shfl_sync(0xffffffffu, run, 31);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        const float hi = static_cast<float>(G[i]);
        sm.g_hi[r] = hi;
        sm.g_lo[r] = static_cast<float>(G[i] - hi);
        sm.beta[r] = bt[i];
        const float eg = expf(hi);
        factors[kFA + r] = -bt[i] * eg * sm.ck[r];
        factors[kFB + r] = bt[i];
        factors[kFQ + r] = eg * sm.cq[r];
        factors[kFW + r] = expf(static_cast<float>(last - G[i])) * sm.ck[r];
      }
      if (lane == 0) factors[kFEnd] = expf(static_cast<float>(last));
    }
    __syncthreads();
    // A into t and P out: eight columns j0 .. j0 + 7 a warp, a row per lane
    const int j0 = w * 8;
    {
#pragma unroll 1
      for (int s = 0; s < 2; ++s) {
        const int i = s * 32 + lane;
        float av[8], pv[8];
        if (j0 < (s + 1) * 32) {
          const float gh = sm.g_hi[i], gl = sm.g_lo[i], bi = sm.beta[i] * sm.ck[i], qi = sm.cq[i];
#pragma unroll
          for (int j4 = 0; j4 < 8; j4 += 4) {
            const float4 h4 = *reinterpret_cast<const float4*>(&sm.g_hi[j0 + j4]);
            const float4 l4 = *reinterpret_cast<const float4*>(&sm.g_lo[j0 + j4]);
            const float4 c4 = *reinterpret_cast<const float4*>(&sm.ck[j0 + j4]);
            const float4 k4 = *reinterpret_cast<const float4*>(&sm.gk[i * kGS + j0 + j4]);
            const float4 q4 = *reinterpret_cast<const float4*>(&sm.gq[i * kGS + j0 + j4]);
            const float hj[4] = {h4.x, h4.y, h4.z, h4.w}, lj[4] = {l4.x, l4.y, l4.z, l4.w},
                        cj[4] = {c4.x, c4.y, c4.z, c4.w}, kj[4] = {k4.x, k4.y, k4.z, k4.w},
                        qj[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int jj = j0 + j4 + j;
              const float f = expf((gh - hj[j]) + (gl - lj[j])) * cj[j];
              pv[j4 + j] = jj <= i ? qj[j] * qi * f : 0.f;
              av[j4 + j] = jj < i ? kj[j] * bi * f : 0.f;
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) av[j] = pv[j] = 0.f;
        }
        *reinterpret_cast<float4*>(&sm.t[i * kGS + j0]) = make_float4(av[0], av[1], av[2], av[3]);
        *reinterpret_cast<float4*>(&sm.t[i * kGS + j0 + 4]) = make_float4(av[4], av[5], av[6], av[7]);
        if (w / 2 <= i / 16) store_terms<2>(pv, dst + kRecBytes + tri_at(i, w));
      }
    }
    __syncthreads();
    invert(sm);
    // T's terms, eight lanes a row
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int i = s * 32 + (tid >> 3), jt = (tid & 7) * 8;
      if (jt / 16 > i / 16) continue;
      float tv[8];
#pragma unroll
      for (int j4 = 0; j4 < 8; j4 += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&sm.t[i * kGS + jt + j4]);
        tv[j4] = v.x; tv[j4 + 1] = v.y; tv[j4 + 2] = v.z; tv[j4 + 3] = v.w;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (jt + j > i) tv[j] = 0.f;
      store_terms<3>(tv, dst + tri_at(i, tid & 7));
    }
    // the next head's sums and decays are written after every thread has read this one's (the inverse's barriers),
    // its A after the barrier behind them
  }
}

}  // namespace

// ------------------------------------------------------------------ host
namespace {

// Chunks are taken in segments of slots, which bounds the workspace.  One sequence: what dn_prep_kernel writes
// should still be in L2 when a walk reads it.  Several: a segment holds whole sequences but for its ends, so it
// has to be long enough for all SMs to have some to walk.
constexpr int64_t kSegmentBytes = int64_t{128} << 20, kBatchSegmentBytes = int64_t{1} << 30;

int64_t slot_bytes(int n_heads, int n_key_heads, int dk) {
  return static_cast<int64_t>(n_key_heads) * 2 * C * dk * 2 + static_cast<int64_t>(n_heads) * kHeadBytes;
}
int64_t segment_slots(int64_t n_seqs, int64_t slots, int n_heads, int n_key_heads, int dk) {
  const int64_t fit = (n_seqs == 1 ? kSegmentBytes : kBatchSegmentBytes) / slot_bytes(n_heads, n_key_heads, dk);
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

// Which walk: the quads' for few states, the warps' for many, whatever their lengths (which only the device knows).
// Blocks come in rounds of one per SM, and a chunk of a block takes, in 0.1 us (one head, from 2048 to 6144 tokens):
// 32 columns in the quads' walk 29 for dk = 128 and 23 for dk = 64, 64 columns in the warps' 50 and 36, 128 columns
// 78 and 54.  Quads against warps, us: 32 / 64 / 128 states of 128 x 128 with 2048 tokens 137 / 210, 266 / 247,
// 522 / 409; 160 with 1000 tokens 334 / 334-354; 512 of 64 x 32 with 1000 tokens 372 / 436.
template <int DK>
bool quad_walk(int64_t states, int dv, int sms) {
  auto rounds = [&](int cols) { return (states * ((dv + cols - 1) / cols) + sms - 1) / sms; };
  const int64_t narrow = rounds(kWarpCols / 2) * (DK == 128 ? 50 : 36), wide = rounds(kWarpCols) * (DK == 128 ? 78 : 54);
  return rounds(kQuadCols) * (DK == 128 ? 29 : 23) <= (narrow < wide ? narrow : wide);
}

template <int DK>
int run(const DnRows& a, const int32_t* cu, int64_t n_seqs, int64_t tokens, const DeviceInfo& dev, void* workspace,
        qfn_stream_t stream) {
  constexpr const char* what = "qfn_deltanet_chunk";
  const int key_heads = a.heads / a.ratio;
  const int64_t slots = tokens / C + n_seqs, seg = segment_slots(n_seqs, slots, a.heads, key_heads, DK);
  const bool quad = quad_walk<DK>(n_seqs * a.heads, a.dv, dev.sm_count);
  const int cols = quad ? kQuadCols : kWarpCols / 2;
  const int64_t blocks = n_seqs * a.heads * ((a.dv + cols - 1) / cols);
  QFN_REQUIRE(blocks <= 0x7fffffff && seg * key_heads <= 0x7fffffff, QFN_ERR_UNSUPPORTED, "%s: too many sequences",
              what);
  auto even = [](const void* p, int64_t row, int64_t head) {   // in pieces of 16 bytes
    return aligned(p, 16) && row % 8 == 0 && head % 8 == 0;
  };
  const bool kq_vec = even(a.q, a.q_row, a.q_head) && even(a.k, a.k_row, a.k_head);
  const bool v_vec = even(a.v, a.v_row, a.v_head);
  // the kernels' shared memory, once for each device
  static std::atomic<uint64_t> prepared{0};
  const uint64_t bit = uint64_t{1} << dev.device;
  cudaError_t e = cudaSuccess;
  if (!(prepared.load(std::memory_order_acquire) & bit)) {
    const cudaFuncAttribute smem = cudaFuncAttributeMaxDynamicSharedMemorySize;
    e = cudaFuncSetAttribute(dn_prep_kernel<DK>, smem, sizeof(PrepSmem<DK>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(dn_walk_quad_kernel<DK>, smem, sizeof(QuadSmem<DK>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(dn_walk_warp_kernel<DK>, smem, sizeof(WarpSmem<DK>));
    if (e != cudaSuccess) return set_error(QFN_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
    prepared.fetch_or(bit, std::memory_order_release);
  }
  const Plan plan{cu, n_seqs, tokens, cu ? 0 : tokens / n_seqs};
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const Work work{ws, ws + seg * key_heads * (2 * C * DK * 2)};
  for (int64_t s0 = 0; s0 < slots && e == cudaSuccess; s0 += seg) {
    const int64_t s1 = s0 + seg < slots ? s0 + seg : slots;
    e = launch(dn_prep_kernel<DK>, (s1 - s0) * key_heads, kPrepThreads, sizeof(PrepSmem<DK>), as_stream(stream), a, plan,
               work, s0, kq_vec);
    if (e == cudaSuccess)
      e = quad ? launch(dn_walk_quad_kernel<DK>, blocks, kQuadThreads, sizeof(QuadSmem<DK>), as_stream(stream), a, plan,
                        work, s0, s1, v_vec)
               : launch(dn_walk_warp_kernel<DK>, blocks, kWarpThreads, sizeof(WarpSmem<DK>), as_stream(stream), a, plan,
                        work, s0, s1, v_vec, dev.sm_count);
  }
  if (e != cudaSuccess) return set_error(QFN_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace

bool dn_chunk_takes(int64_t longest, int64_t n_seqs, int n_heads, int dk, int dv) {
  const bool few = n_seqs * n_heads * (dv / 32) <= 300;   // blocks of the recurrence: up to two an SM
  const int64_t by_size = 8 + 65536 / (static_cast<int64_t>(dk) * dv);
  return dk <= 128 && longest > (few || by_size < 10 ? 10 : by_size < 24 ? by_size : 24);
}

size_t dn_chunk_workspace(int64_t tokens, int64_t n_seqs, int n_heads, int n_key_heads, int dk) {
  const int64_t slots = tokens / C + n_seqs;
  return static_cast<size_t>(segment_slots(n_seqs, slots, n_heads, n_key_heads, dk) * slot_bytes(n_heads, n_key_heads, dk));
}

int dn_chunk(const DnRows& a, const int32_t* cu, int64_t n_seqs, int64_t tokens, int dk, const DeviceInfo& dev,
             void* workspace, qfn_stream_t stream) {
  return dk == 64 ? run<64>(a, cu, n_seqs, tokens, dev, workspace, stream)
                  : run<128>(a, cu, n_seqs, tokens, dev, workspace, stream);
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
