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
constexpr int kSorted = 64;        // sequences up to which the longest are walked first
constexpr int kOutStages = 2;    // chunks of what only the outputs read
constexpr int kPrepThreads = 256;
constexpr int kThreads = 12 * 32; // 8 warps of the recurrence, 4 of the outputs and the copies
constexpr int kGS = 68;          // row pitch of the 64 x 64 fp32 matrices of dn_prep_kernel

// Per chunk and value head: T hi, T lo (f16, 128-byte rows, swizzled), the
// tokens' factors and the chunk's scales, then P (as T).
constexpr int kMat = C * C * 2;
enum { kFA = 0, kFB = C, kFQ = 2 * C, kFW = 3 * C, kFEnd = 4 * C };   // -beta e^G ck, beta, e^G cq, e^(G64 - G) ck
// + e^G64, scale of T, scale of P, largest row sums of e^(G64 - G) ck |T| and of |T|, largest |beta| e^G
constexpr int kFactors = 4 * C + 8;
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

// max(m, |a|, |b|), NaN dropped or kept
__device__ __forceinline__ float max_abs(float m, float a, float b) {
  asm("max.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float max_abs_nan(float m, float a, float b) {
  asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(a), "f"(b));
  return m;
}

// D += A B and, for the first product of an accumulator, D = A B.  Not volatile: the compiler may
// move the products between the loads.
__device__ __forceinline__ void mma_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Byte offset of 16-byte piece `ch` of row `row` in a matrix of ROW-byte rows
// whose pieces are permuted so that eight rows' equal pieces lie in distinct banks.
template <int ROW>
__device__ __forceinline__ uint32_t swz(int row, int ch) {
  return static_cast<uint32_t>(row * ROW + ((ROW == 64 ? ch ^ ((row >> 1) & 3) : ch ^ (row & 7)) << 4));
}

// ------------------------------------------------------------------ what needs no state
template <int DK>
struct PrepSmem {
  union {
    struct {
      unsigned char k[C * DK * 2], q[C * DK * 2];   // f16 rows, swizzled
    };
    struct {
      float t[C * kGS];     // A, then T
      float y[32 * 36];     // A21 T11
    };
  };
  float gk[C * kGS], gq[C * kGS];   // k_i . k_j, q_i . k_j of the scaled rows
  float g_hi[C], g_lo[C], ck[C], cq[C], beta[C], w[C];
  uint32_t red[3][kPrepThreads / 32];
  float p_scale;
};

// The inverse of I + A, A strictly lower triangular in t, in fp32: the two 32 x 32 halves of the
// diagonal by substitution, a column per lane, then T21 = -T22 (A21 T11) by the whole block.
template <int DK>
__device__ __forceinline__ void invert(PrepSmem<DK>& sm) {
  const int tid = threadIdx.x, w = tid >> 5, c = tid & 31;
  if (w < 2) {
    float* t = sm.t + w * 32 * (kGS + 1);
    float x[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
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
    for (int i = 0; i < 32; ++i) t[i * kGS + c] = x[i];
  }
  __syncthreads();
  // a thread: row r, columns c4 .. c4 + 3
  const int r = tid >> 3, c4 = (tid & 7) * 4;
  auto product = [&](const float* row, const float* m, int pitch) {
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int k = 0; k < 32; k += 4) {
      const float4 av = *reinterpret_cast<const float4*>(row + k);
      const float ak[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 b = *reinterpret_cast<const float4*>(m + (k + i) * pitch + c4);
        y.x = fmaf(ak[i], b.x, y.x); y.y = fmaf(ak[i], b.y, y.y); y.z = fmaf(ak[i], b.z, y.z); y.w = fmaf(ak[i], b.w, y.w);
      }
    }
    return y;
  };
  *reinterpret_cast<float4*>(&sm.y[r * 36 + c4]) = product(sm.t + (32 + r) * kGS, sm.t, kGS);
  __syncthreads();
  const float4 y = product(sm.t + (32 + r) * kGS + 32, sm.y, 36);
  *reinterpret_cast<float4*>(&sm.t[(32 + r) * kGS + c4]) = make_float4(-y.x, -y.y, -y.z, -y.w);
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

// Eight lanes hold a bf16 row of q or k: as f16 after a power-of-two scale 2^e (bf16 is exact in f16 then) to
// shared memory and to the workspace, both swizzled; the row's factor (1 / norm) 2^-e.
template <int DK>
__device__ __forceinline__ void f16_row(const uint4 (&x)[DK / 64], unsigned char* tile, unsigned char* copy, int row,
                                        float* factor, float divide) {
  const int part = threadIdx.x & 7;
  constexpr int N = DK / 8;
  float v[N], ss[2] = {0.f, 0.f}, m[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < DK / 64; ++i) {
    const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[i * 8 + 2 * j] = __uint_as_float(u[j] << 16);
      v[i * 8 + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    ss[i & 1] = fmaf(v[i], v[i], ss[i & 1]);
    m[i & 1] = fmaxf(m[i & 1], fabsf(v[i]));
  }
  float s = ss[0] + ss[1], mm = fmaxf(m[0], m[1]);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  }
  const int e = scale_exp(__float_as_uint(mm));
  const float sc = exp2i(e);
#pragma unroll
  for (int i = 0; i < DK / 64; ++i) {
    const uint4 h = make_uint4(pack_h2(v[i * 8] * sc, v[i * 8 + 1] * sc), pack_h2(v[i * 8 + 2] * sc, v[i * 8 + 3] * sc),
                               pack_h2(v[i * 8 + 4] * sc, v[i * 8 + 5] * sc), pack_h2(v[i * 8 + 6] * sc, v[i * 8 + 7] * sc));
    const uint32_t at = swz<DK * 2>(row, part * (DK / 64) + i);
    *reinterpret_cast<uint4*>(tile + at) = h;
    *reinterpret_cast<uint4*>(copy + at) = h;
  }
  // a row of zeros counts for nothing: its factor, up to 1000, would take the others' digits
  if (part == 0) *factor = s == 0.f ? 0.f : rsqrtf(s + 1e-6f) / divide * exp2i(-e);
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
    n = min(slot * C / (plan.tokens / plan.n_seqs + C), plan.n_seqs - 1);
    while (n + 1 < plan.n_seqs && plan.slot(n + 1) <= slot) ++n;
  }
  const int64_t t0 = plan.begin(n) + (slot - plan.slot(n)) * C;
  const int cnt = static_cast<int>(min(static_cast<int64_t>(C), plan.end(n) - t0));
  if (cnt <= 0) return;

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
      f16_row<DK>(x[i], i < 2 ? sm.k : sm.q, copy + (i < 2 ? 0 : C * DK * 2), r, i < 2 ? &sm.ck[r] : &sm.cq[r],
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
    float* factors = reinterpret_cast<float*>(dst + 2 * kMat);
    // Running sum of g in 64 bits, kept as two floats: differences of far tokens' sums keep their
    // digits.  exp(-200) is 0 in fp32, and a finite sum keeps exp(G_i - G_j) a number.
    if (w == 0) {
      double s[2];
      float bt[2], rise = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        const float gv = r < cnt ? a.g[(t0 + r) * a.g_row + h * a.g_head] : 0.f;
        rise += fmaxf(gv, 0.f);
        s[i] = gv < -200.f ? -200.f : gv;
        bt[i] = r < cnt ? bf16_bits_to_f32(a.beta[(t0 + r) * a.b_row + h * a.b_head]) : 0.f;
      }
      double run = s[0] + s[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      rise = warp_sum(rise);
      float bmax = 0.f;
      const double G[2] = {run - s[1], run};
      const double last = __shfl_sync(0xffffffffu, run, 31);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        const float hi = static_cast<float>(G[i]);
        sm.g_hi[r] = hi;
        sm.g_lo[r] = static_cast<float>(G[i] - hi);
        sm.beta[r] = bt[i];
        const float eg = expf(hi), wt = expf(static_cast<float>(last - G[i])) * sm.ck[r];
        sm.w[r] = wt;
        bmax = fmaxf(bmax, fabsf(bt[i]) * eg);
        factors[kFA + r] = -bt[i] * eg * sm.ck[r];
        factors[kFB + r] = bt[i];
        factors[kFQ + r] = eg * sm.cq[r];
        factors[kFW + r] = wt;
      }
      bmax = __uint_as_float(__reduce_max_sync(0xffffffffu, finite_bits(bmax)));
      if (lane == 0) {
        factors[kFEnd + 5] = bmax;
        // |q_i . k_j| <= 1 / q_scale after the norms, and no decay is above the sum of the rises
        const float bound = expf(rise) / a.q_scale * 1.01f;
        const int e = bound < 0x1p127f ? scale_exp(__float_as_uint(bound)) : -112;
        sm.p_scale = exp2i(e);
        factors[kFEnd] = expf(static_cast<float>(last));
        factors[kFEnd + 2] = exp2i(-e);
      }
    }
    __syncthreads();
    // A into t and P out: eight columns j0 .. j0 + 7 a warp, a row per lane
    const int j0 = w * 8;
    {
      const float psc = sm.p_scale;
#pragma unroll 1
      for (int s = 0; s < 2; ++s) {
        const int i = s * 32 + lane;
        float av[8], pv[8];
        if (j0 < (s + 1) * 32) {
          const float gh = sm.g_hi[i], gl = sm.g_lo[i], bi = sm.beta[i] * sm.ck[i], qi = sm.cq[i] * psc;
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
              pv[j4 + j] = jj <= i ? f * qi * qj[j] : 0.f;
              av[j4 + j] = jj < i ? f * bi * kj[j] : 0.f;
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) av[j] = pv[j] = 0.f;
        }
        *reinterpret_cast<float4*>(&sm.t[i * kGS + j0]) = make_float4(av[0], av[1], av[2], av[3]);
        *reinterpret_cast<float4*>(&sm.t[i * kGS + j0 + 4]) = make_float4(av[4], av[5], av[6], av[7]);
        *reinterpret_cast<uint4*>(dst + kRecBytes + swz<128>(i, w)) =
            make_uint4(pack_h2(pv[0], pv[1]), pack_h2(pv[2], pv[3]), pack_h2(pv[4], pv[5]), pack_h2(pv[6], pv[7]));
      }
    }
    __syncthreads();
    invert(sm);
    // T's scale, and a bound of the weighted d for the walk: the largest row sum of w |T| (eight lanes a row)
    float tv[2][8];
    uint32_t tm = 0, wm = 0, top = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int i = s * 32 + (tid >> 3), jt = (tid & 7) * 8;
      float sum = 0.f;
#pragma unroll
      for (int j4 = 0; j4 < 8; j4 += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&sm.t[i * kGS + jt + j4]);
        tv[s][j4] = v.x; tv[s][j4 + 1] = v.y; tv[s][j4 + 2] = v.z; tv[s][j4 + 3] = v.w;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (jt + j > i) tv[s][j] = 0.f;
        const uint32_t b = finite_bits(tv[s][j]);
        tm = max(tm, b);
        sum += __uint_as_float(b);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      wm = max(wm, finite_bits(sum * sm.w[i]));
      top = max(top, finite_bits(sum));
    }
    tm = __reduce_max_sync(0xffffffffu, tm);
    wm = __reduce_max_sync(0xffffffffu, wm);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) {
      sm.red[0][w] = tm;
      sm.red[1][w] = wm;
      sm.red[2][w] = top;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPrepThreads / 32; ++i) {
      tm = max(tm, sm.red[0][i]);
      wm = max(wm, sm.red[1][i]);
      top = max(top, sm.red[2][i]);
    }
    const int et = scale_exp(tm);
    const float sc = exp2i(et);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) split2(tv[s][2 * j] * sc, tv[s][2 * j + 1] * sc, hi[j], lo[j]);
      const uint32_t at = swz<128>(s * 32 + (tid >> 3), tid & 7);
      *reinterpret_cast<uint4*>(dst + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(dst + kMat + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    if (tid == 0) {
      factors[kFEnd + 1] = exp2i(-et);
      factors[kFEnd + 3] = __uint_as_float(wm) * 1.0001f;   // the sum's own rounding
      factors[kFEnd + 4] = __uint_as_float(top) * 1.0001f;
    }
    // the next head's factors overwrite this one's only after every thread has passed the barrier above,
    // its A only after the next one
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
  uint4 s_hi[2][2][4][DK / 64][32];   // [buffer][columns][quarter of dk][k tile][lane]
  uint4 d_hi[2][2][4][32];            // [buffer][columns][token block][lane]
  float4 x[2][4][3][2][32];           // partial S^T k [columns][quarter][block - quarter - 1][tile][lane]
  uint4 rx[2][4][2][32];              // R [columns][token block][hi, lo][lane]
  uint4 dx[2][4][2][32];              // weighted d, likewise
  int bad[2][2][16];                  // [buffer][columns][column] first token whose R is not finite, or C
  float s_inv[2][2], d_inv[2][2];     // [buffer][columns]
  float s_max[2][4], v_max[2][4];     // [columns][quarter]
  uint64_t full[kStages], empty[kStages], out_full[kOutStages], out_empty[kOutStages];
  int length[kSorted], seq;
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

// The four warps of 16 columns.
__device__ __forceinline__ void quad_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, 128;" ::"r"(id + 1) : "memory");
}

// Largest finite magnitude of a warp's values, the same in every lane.
template <int N>
__device__ __forceinline__ float warp_max(const float (&v)[N][4]) {
  float m0 = 0.f, m1 = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m0 = max_abs(m0, v[i][0], v[i][1]);
    m1 = max_abs(m1, v[i][2], v[i][3]);
  }
  uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(m0, m1)));
  if (b >= 0x7f800000u) {   // an infinity somewhere: the other columns keep their own scale
    b = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) b = max(b, finite_bits(v[i][j]));
    b = __reduce_max_sync(0xffffffffu, b);
  }
  return __uint_as_float(b);
}

// Power-of-two scale for a bound; not finite: the smallest scale.
__device__ __forceinline__ int bound_exp(float bound) {
  return bound < 0x1p127f ? scale_exp(__float_as_uint(bound)) : -112;
}

// Accumulators of two neighbouring 16 x 8 tiles as the hi and lo fragments of a 16 x 16 operand.
__device__ __forceinline__ void frag_split(const float (&a)[4], const float (&b)[4], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  split2(a[0], a[1], hi[0], lo[0]);
  split2(a[2], a[3], hi[1], lo[1]);
  split2(b[0], b[1], hi[2], lo[2]);
  split2(b[2], b[3], hi[3], lo[3]);
}

__device__ __forceinline__ uint4 as_uint4(const uint32_t (&r)[4]) { return make_uint4(r[0], r[1], r[2], r[3]); }
__device__ __forceinline__ void from_uint4(uint32_t (&r)[4], uint4 v) { r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w; }

// The output warps of 16 columns take blocks of 16 tokens so that their triangular products take
// the same time: 0 and 3 to one, 1 and 2 to the other.
__device__ __forceinline__ int block_of(int half, int i) { return half ? 1 + i : 3 * i; }

// A block's values of a lane's columns g (first token bad0) and g + 8 (bad1) from those tokens on become v.
__device__ __forceinline__ void spoil(float* d, int block, int bad0, int bad1, float v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int tok = block * 16 + i * 8 + 2 * (threadIdx.x & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (tok + (j & 1) >= (j < 2 ? bad0 : bad1)) d[i * 4 + j] = v;
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
  int64_t seq = blockIdx.x / cb / a.heads;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 129);   // the bulk copies' bytes, 128 lanes' copies of v
      mbar_init(&sm.empty[i], 12);
    }
    for (int i = 0; i < kOutStages; ++i) {
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
  const bool ok = !plan.cu || dn_plan_ok(plan.cu, plan.n_seqs, plan.tokens);
  // Blocks start in order and a sequence's walk cannot be split, so the longest go first: block n takes the
  // sequence with n longer ones (equal ones in their order).  Worth its n_seqs^2 reads for few sequences only.
  if (ok && plan.cu && plan.n_seqs <= kSorted) {
    const int n = static_cast<int>(plan.n_seqs);
    if (tid < n) sm.length[tid] = plan.cu[tid + 1] - plan.cu[tid];
    __syncthreads();
    if (tid < n) {
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += sm.length[i] > sm.length[tid] || (sm.length[i] == sm.length[tid] && i < tid);
      if (rank == seq) sm.seq = tid;
    }
    __syncthreads();
    seq = sm.seq;
  }
  __syncthreads();
  // this launch's chunks of the sequence
  const int64_t begin = ok ? plan.begin(seq) : 0, base = ok ? plan.slot(seq) : slot0;
  const int64_t len = ok ? plan.end(seq) - begin : 0, chunks = (len + C - 1) / C;
  const int64_t first = max(slot0 - base, static_cast<int64_t>(0)), last = min(slot1 - base, chunks);
  if (base >= slot1 || (first > 0 && first >= last)) return;
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
    float S[NT][4];   // S^T 2^e: rows are columns g and g + 8, columns are dk
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
    float acc[8][4], vb[2][4];   // this quarter's part of S^T k 2^e, blocks qd, qd + 1, .. (mod 4); beta v of the block
    float inv = 1.f;             // 2^-e
    uint32_t kx[KT][4][4];       // k's fragments of the chunk that comes next
    auto load_keys = [&](uint32_t n) {
      wait(&sm.full[n % kStages], (n / kStages) & 1);
      const uint32_t kb = smem_u32(sm.stage[n % kStages].k);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          ldsm4(kx[kt][b], kb + swz<DK * 2>(((qd + b) & 3) * 16 + (lane & 7) + ((lane >> 4) << 3),
                                            d0 / 8 + kt * 2 + ((lane >> 3) & 1)));
    };
    // S as f16 terms times the keys of chunk n; the hi terms go to the warps of the outputs too.  What chunk
    // n's R needs besides comes behind the products.
    auto times_keys = [&](uint32_t n) {
      const uint32_t bf = n & 1;
      const Stage<DK>& sn = sm.stage[n % kStages];
      uint32_t hi[KT][4], lo[KT][4];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) frag_split(S[2 * kt], S[2 * kt + 1], hi[kt], lo[kt]);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (kt == 0) {
            mma_first(acc[2 * b], hi[kt], kx[kt][b][0], kx[kt][b][1]);
            mma_first(acc[2 * b + 1], hi[kt], kx[kt][b][2], kx[kt][b][3]);
          } else {
            mma_add(acc[2 * b], hi[kt], kx[kt][b][0], kx[kt][b][1]);
            mma_add(acc[2 * b + 1], hi[kt], kx[kt][b][2], kx[kt][b][3]);
          }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          mma_add(acc[2 * b], lo[kt], kx[kt][b][0], kx[kt][b][1]);
          mma_add(acc[2 * b + 1], lo[kt], kx[kt][b][2], kx[kt][b][3]);
        }
      }
      if (n >= 2) wait(&sm.out_done[bf][grp], ((n >> 1) + 1) & 1);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) sm.s_hi[bf][grp][qd][kt][lane] = as_uint4(hi[kt]);
      if (qd == 0) {
        if (lane == 0) sm.s_inv[bf][grp] = inv;
        if (lane < 16) sm.bad[bf][grp][lane] = C;
      }
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
      const float s_max = warp_max(S) * inv, v_max = warp_max(vb);
      if (lane == 0) {
        sm.s_max[grp][qd] = s_max;
        sm.v_max[grp][qd] = v_max;
      }
    };
    auto largest = [](const float (&v)[4]) {
      const float4 x = *reinterpret_cast<const float4*>(v);
      return fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
    };
    if (first < last) {
      const float m = warp_max(S);
      if (lane == 0) sm.s_max[grp][qd] = m;
      quad_sync(grp);
      const int e = scale_exp(__float_as_uint(largest(sm.s_max[grp])));
      quad_sync(grp);   // s_max is written again below
      const float s = exp2i(e);
      inv = exp2i(-e);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) S[i][j] *= s;
      load_keys(0);
      times_keys(0);
    }
    for (int64_t ci = first; ci < last; ++ci) {
      const uint32_t it = static_cast<uint32_t>(ci - first), st = it % kStages, buf = it & 1;
      Stage<DK>& sg = sm.stage[st];
      const uint32_t kb = smem_u32(sg.k);
      const bool more = ci + 1 < last;
      const float4 fe = *reinterpret_cast<const float4*>(&sg.f[kFEnd]);
      const float2 fm = *reinterpret_cast<const float2*>(&sg.f[kFEnd + 4]);
      // the quarters' parts meet, each in the warp of its token block
#pragma unroll
      for (int b = 1; b < 4; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          sm.x[grp][qd][b - 1][j][lane] = make_float4(acc[2 * b + j][0], acc[2 * b + j][1], acc[2 * b + j][2], acc[2 * b + j][3]);
      quad_sync(grp);
      float R[2][4];
      const float s_all = largest(sm.s_max[grp]);
      // |k| <= 1: S^T k is at most sqrt(dk) times S's largest
      const float r_bound = fmaf(fm.y * (DK == 128 ? 11.4f : 8.1f), s_all, largest(sm.v_max[grp]));
      const int re = bound_exp(r_bound);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 o1 = sm.x[grp][(qd + 1) & 3][2][j][lane];
        const float4 o2 = sm.x[grp][(qd + 2) & 3][1][j][lane];
        const float4 o3 = sm.x[grp][(qd + 3) & 3][0][j][lane];
        const float2 fa = *reinterpret_cast<const float2*>(&sg.f[kFA + qd * 16 + j * 8 + 2 * t]);
        const float ax = fa.x * inv, ay = fa.y * inv;
        R[j][0] = fmaf(ax, (acc[j][0] + o1.x) + (o2.x + o3.x), vb[j][0]);
        R[j][1] = fmaf(ay, (acc[j][1] + o1.y) + (o2.y + o3.y), vb[j][1]);
        R[j][2] = fmaf(ax, (acc[j][2] + o1.z) + (o2.z + o3.z), vb[j][2]);
        R[j][3] = fmaf(ay, (acc[j][3] + o1.w) + (o2.w + o3.w), vb[j][3]);
      }
      const float r_nan = max_abs_nan(max_abs_nan(max_abs_nan(max_abs_nan(0.f, R[0][0], R[0][1]), R[0][2], R[0][3]), R[1][0],
                                                  R[1][1]), R[1][2], R[1][3]);
      if (__any_sync(0xffffffffu, !(r_nan < CUDART_INF_F))) {
        // A token's infinity or NaN may not reach the tokens before it through T's and P's zeros:
        // it is taken out here and put back into d from that token on.
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!(fabsf(R[i][j]) < CUDART_INF_F)) {
              atomicMin(&sm.bad[buf][grp][g + (j >> 1) * 8], qd * 16 + i * 8 + 2 * t + (j & 1));
              R[i][j] = 0.f;
            }
      }
      uint32_t rh[4], rl[4];
      {
        const float s = exp2i(re);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) R[i][j] *= s;
        frag_split(R[0], R[1], rh, rl);
        sm.rx[grp][qd][0][lane] = as_uint4(rh);
        sm.rx[grp][qd][1][lane] = as_uint4(rl);
      }
      // T's rows of this block; beyond the diagonal they are zero, and all four warps go the same way
      uint32_t yh[4][4], yl[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t at = swz<128>(qd * 16 + (lane & 7) + ((lane >> 4) << 3), ((qd + j) & 3) * 2 + ((lane >> 3) & 1));
        ldsm4(yh[j], smem_u32(sg.t_hi) + at);
        ldsm4(yl[j], smem_u32(sg.t_lo) + at);
      }
      quad_sync(grp);
      // d = T R of this block: source blocks qd, qd + 1, .. (mod 4), in two sets of accumulators
      float p[2][2][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t xh[4], xl[4];
        if (j == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) { xh[i] = rh[i]; xl[i] = rl[i]; }
        } else {
          from_uint4(xh, sm.rx[grp][(qd + j) & 3][0][lane]);
          from_uint4(xl, sm.rx[grp][(qd + j) & 3][1][lane]);
        }
        float(&d0_)[4] = p[j & 1][0];
        float(&d1_)[4] = p[j & 1][1];
        if (j < 2) {
          mma_first(d0_, xh, yh[j][0], yh[j][1]);
          mma_first(d1_, xh, yh[j][2], yh[j][3]);
        } else {
          mma_add(d0_, xh, yh[j][0], yh[j][1]);
          mma_add(d1_, xh, yh[j][2], yh[j][3]);
        }
        mma_add(d0_, xl, yh[j][0], yh[j][1]);
        mma_add(d1_, xl, yh[j][2], yh[j][3]);
        mma_add(d0_, xh, yl[j][0], yl[j][1]);
        mma_add(d1_, xh, yl[j][2], yl[j][3]);
      }
      // k^T's fragments for the state's update
      uint32_t kt_[4][NT / 2][4];
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int np = 0; np < NT / 2; ++np)
          ldsm4t(kt_[b][np], kb + swz<DK * 2>(((qd + b) & 3) * 16 + (lane & 15), d0 / 8 + np * 2 + (lane >> 4)));
      // d's scales come from bounds: R's times T's row sums, weighted (for the state, in two terms) and not
      // (for the outputs, in one)
      const float w_bound = r_bound * fe.w;
      const int we = bound_exp(w_bound), de = bound_exp(r_bound * fm.x);
      const float d_inv = w_bound > 0.f ? exp2i(-we) : 0.f;
      const float c = exp2i(-re) * fe.y, c16 = c * exp2i(de), cw = c * exp2i(we);
      const int bad0 = sm.bad[buf][grp][g], bad1 = sm.bad[buf][grp][g + 8];
      const bool any_bad = __any_sync(0xffffffffu, bad0 < C || bad1 < C);
      uint32_t wh[4], wl[4], d16[4];
      {
        float d[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) d[i][j] = p[0][i][j] + p[1][i][j];
        if (any_bad) spoil(&d[0][0], qd, bad0, bad1, 0.f);
        d16[0] = pack_h2(d[0][0] * c16, d[0][1] * c16);
        d16[1] = pack_h2(d[0][2] * c16, d[0][3] * c16);
        d16[2] = pack_h2(d[1][0] * c16, d[1][1] * c16);
        d16[3] = pack_h2(d[1][2] * c16, d[1][3] * c16);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 fw = *reinterpret_cast<const float2*>(&sg.f[kFW + qd * 16 + i * 8 + 2 * t]);
          const float wx = fw.x * cw, wy = fw.y * cw;
          d[i][0] *= wx;
          d[i][1] *= wy;
          d[i][2] *= wx;
          d[i][3] *= wy;
        }
        if (any_bad) spoil(&d[0][0], qd, bad0, bad1, CUDART_NAN_F);
        frag_split(d[0], d[1], wh, wl);
        sm.dx[grp][qd][0][lane] = as_uint4(wh);
        sm.dx[grp][qd][1][lane] = as_uint4(wl);
      }
      quad_sync(grp);
      // S = e^G64 S + d k^T for this quarter of dk.  Its scale comes from a bound: 64 products of d and
      // k, both below 2^15 as f16.
      const int e = bound_exp(fmaf(s_all, fe.x, d_inv * 0x1p36f));
      const float s = exp2i(e), keep = fe.x * inv * s, gain = d_inv * s;
      inv = exp2i(-e);
      {
        float u[NT][4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t xh[4], xl[4];
          if (b == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { xh[i] = wh[i]; xl[i] = wl[i]; }
          } else {
            from_uint4(xh, sm.dx[grp][(qd + b) & 3][0][lane]);
            from_uint4(xl, sm.dx[grp][(qd + b) & 3][1][lane]);
          }
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            const uint32_t(&y)[4] = kt_[b][np];
            if (b == 0) {
              mma_first(u[2 * np], xh, y[0], y[1]);
              mma_first(u[2 * np + 1], xh, y[2], y[3]);
            } else {
              mma_add(u[2 * np], xh, y[0], y[1]);
              mma_add(u[2 * np + 1], xh, y[2], y[3]);
            }
          }
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            mma_add(u[2 * np], xl, kt_[b][np][0], kt_[b][np][1]);
            mma_add(u[2 * np + 1], xl, kt_[b][np][2], kt_[b][np][3]);
          }
        }
        if (more) load_keys(it + 1);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) S[i][j] = fmaf(u[i][j], gain, S[i][j] * keep);
      }
      // d for the outputs of this chunk
      sm.d_hi[buf][grp][qd][lane] = make_uint4(d16[0], d16[1], d16[2], d16[3]);
      if (qd == 0 && lane == 0) sm.d_inv[buf][grp] = exp2i(-de);
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.d_full[buf][grp]);
        mbar_arrive(&sm.empty[st]);
      }
      if (more) times_keys(it + 1);
    }
    float* dst = a.s_out + s_at + grp * 16 + g;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int64_t r = static_cast<int64_t>(d0 + i * 8 + 2 * t) * a.dv;
      dst[r] = S[i][0] * inv;
      dst[r + a.dv] = S[i][1] * inv;
      dst[r + 8] = S[i][2] * inv;
      dst[r + a.dv + 8] = S[i][3] * inv;
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
      Stage<DK>& sg = sm.stage[it % kStages];
      uint64_t* bar = &sm.full[it % kStages];
      const int64_t t0 = begin + (first + it) * C;
      const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
      if (hl == 0) {
        mbar_arrive_expect_tx(bar, C * DK * 2 + kRecBytes);
        bulk_g2s(sg.k, keys_at(it), C * DK * 2, bar);
        bulk_g2s(sg.t_hi, head_at(it), kRecBytes, bar);
      }
      __syncwarp();
      const uint16_t* v = a.v + t0 * a.v_row + h * a.v_head + c0;
#pragma unroll
      for (int i = 0; i < C * kCols * 2 / 16 / 128; ++i) {
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
      OutStage<DK>& og = sm.out_stage[it % kOutStages];
      uint64_t* bar = &sm.out_full[it % kOutStages];
      if (hl == 0) {
        mbar_arrive_expect_tx(bar, C * DK * 2 + kMat);
        bulk_g2s(og.q, keys_at(it) + C * DK * 2, C * DK * 2, bar);
        bulk_g2s(og.p, head_at(it) + kRecBytes, kMat, bar);
      }
      __syncwarp();
    };
    for (uint32_t i = 0; i < n && i < kStages; ++i) copy_in(i);
    for (uint32_t i = 0; i < n && i < kOutStages; ++i) copy_out_operands(i);
    for (uint32_t it = 0; it < n; ++it) {
      const uint32_t st = it % kStages, so = it % kOutStages, buf = it & 1;
      Stage<DK>& sg = sm.stage[st];
      OutStage<DK>& og = sm.out_stage[so];
      const int64_t t0 = begin + (first + it) * C;
      const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
      wait(&sm.full[st], (it / kStages) & 1);
      wait(&sm.out_full[so], (it / kOutStages) & 1);
      wait(&sm.s_full[buf][grp], (it >> 1) & 1);
      const uint32_t qb = smem_u32(og.q), pb = smem_u32(og.p);
      float acc[4][4], o[4][4];
#pragma unroll
      for (int kt = 0; kt < DK / 16; ++kt) {
        uint32_t x[4];
        from_uint4(x, sm.s_hi[buf][grp][kt / KT][kt % KT][lane]);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t y[4];
          ldsm4(y, qb + swz<DK * 2>(block_of(half, b) * 16 + (lane & 7) + ((lane >> 4) << 3), kt * 2 + ((lane >> 3) & 1)));
          if (kt == 0) {
            mma_first(acc[2 * b], x, y[0], y[1]);
            mma_first(acc[2 * b + 1], x, y[2], y[3]);
          } else {
            mma_add(acc[2 * b], x, y[0], y[1]);
            mma_add(acc[2 * b + 1], x, y[2], y[3]);
          }
        }
      }
      const float si = sm.s_inv[buf][grp];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = *reinterpret_cast<const float2*>(&sg.f[kFQ + block_of(half, i >> 1) * 16 + (i & 1) * 8 + 2 * t]);
        const float fx = f.x * si, fy = f.y * si;
        o[i][0] = acc[i][0] * fx;
        o[i][1] = acc[i][1] * fy;
        o[i][2] = acc[i][2] * fx;
        o[i][3] = acc[i][3] * fy;
      }
      wait(&sm.d_full[buf][grp], (it >> 1) & 1);
      const float ps = sm.d_inv[buf][grp] * sg.f[kFEnd + 2];
#pragma unroll
      for (int bj = 0; bj < 4; ++bj) {   // P is zero beyond the diagonal
        uint32_t x[4];
        from_uint4(x, sm.d_hi[buf][grp][bj][lane]);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t y[4];
          ldsm4(y, pb + swz<128>(block_of(half, b) * 16 + (lane & 7) + ((lane >> 4) << 3), bj * 2 + ((lane >> 3) & 1)));
          if (bj == 0) {
            mma_first(acc[2 * b], x, y[0], y[1]);
            mma_first(acc[2 * b + 1], x, y[2], y[3]);
          } else {
            mma_add(acc[2 * b], x, y[0], y[1]);
            mma_add(acc[2 * b + 1], x, y[2], y[3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = fmaf(acc[i][j], ps, o[i][j]);
      {
        const int bad0 = sm.bad[buf][grp][g], bad1 = sm.bad[buf][grp][g + 8];
        if (__any_sync(0xffffffffu, bad0 < C || bad1 < C)) {
          spoil(&o[0][0], block_of(half, 0), bad0, bad1, CUDART_NAN_F);
          spoil(&o[2][0], block_of(half, 1), bad0, bad1, CUDART_NAN_F);
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
      if (it + kOutStages < n) {
        wait(&sm.out_empty[so], (it / kOutStages) & 1);
        copy_out_operands(it + kOutStages);
      }
      if (it + kStages < n) {
        wait(&sm.empty[st], (it / kStages) & 1);
        copy_in(it + kStages);
      }
    }
    // nothing of these warps may still be on its way when the block ends
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
  const bool kq_vec = even(a.q, a.q_row, a.q_head, 8) && even(a.k, a.k_row, a.k_head, 8);
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
