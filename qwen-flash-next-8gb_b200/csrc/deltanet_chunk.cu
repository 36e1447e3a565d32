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
// each token.  dn_walk_kernel then walks a sequence's chunks, a block per
// (sequence, value head, 128 columns of S), its products on tcgen05.
//
// Precision.  S leaves as fp32, so its factors need more than f16's 11 bits:
// every operand of an S or d product that is not exact is split into two f16
// terms (22 bits) after a power-of-two scale of its column; k and q rows are
// bf16 and exact in f16 after theirs.  The products that only reach the bf16
// output (P d and S^T q) take one term.
#include "deltanet_batch.cuh"
#include "deltanet_chunk.cuh"

namespace qfn {
namespace {

constexpr int C = 64;            // tokens of a chunk
constexpr int kCols = 128;       // state columns of a block: the lanes of TMEM
constexpr int kStages = 3;
constexpr int kPrepThreads = 256;
constexpr int kThreads = 14 * 32; // 8 warps of the recurrence, 4 of the outputs, the MMAs, the copies
constexpr int kGS = 68;          // row pitch of the 64 x 64 fp32 matrices of dn_prep_kernel

// Per chunk and value head: T hi, T lo (f16, 128-byte rows, swizzled), the
// tokens' factors and the chunk's scales, then P (as T).
constexpr int kMat = C * C * 2;
enum { kFA = 0, kFB = C, kFQ = 2 * C, kFW = 3 * C, kFEnd = 4 * C };   // -beta e^G ck, beta, e^G cq, e^(G64 - G) ck
// + e^G64, scale of T, scale of P, largest row sums of e^(G64 - G) ck |T| and of |T|
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

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Byte offset of 16-byte piece `ch` of row `row` in a matrix of 128-byte rows
// in the 128-byte swizzle that tcgen05 reads.
__device__ __forceinline__ uint32_t swz(int row, int ch) {
  return static_cast<uint32_t>(row * 128 + ((ch ^ (row & 7)) << 4));
}

// A k or q tile: pieces of 64 elements of dk side by side, each [64 tokens][128 bytes], swizzled.
__device__ __forceinline__ uint32_t tile_at(int row, int ch) { return (ch >> 3) * (C * 128) + swz(row, ch & 7); }

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
    const uint32_t at = tile_at(row, part * (DK / 64) + i);
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
      ldsm4(x, rows + tile_at(m * 16 + (lane & 15), kt * 2 + (lane >> 4)));
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        if (np > m) continue;
        uint32_t b[4];
        ldsm4(b, cols + tile_at(np * 16 + (lane & 7) + ((lane >> 4) << 3), kt * 2 + ((lane >> 3) & 1)));
        mma_16816(acc[2 * np], x, b[0], b[1]);
        mma_16816(acc[2 * np + 1], x, b[2], b[3]);
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
        factors[kFA + r] = -bt[i] * eg * sm.ck[r];
        factors[kFB + r] = bt[i];
        factors[kFQ + r] = eg * sm.cq[r];
        factors[kFW + r] = wt;
      }
      if (lane == 0) {
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
        *reinterpret_cast<uint4*>(dst + kRecBytes + swz(i, w)) =
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
      const uint32_t at = swz(s * 32 + (tid >> 3), tid & 7);
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
//
// A lane of TMEM is a column of S, so every product is transposed: A holds S^T,
// R^T or d^T as f16 terms in TMEM (K: dk or tokens), B the k, q, T or P tile
// in shared memory (N: tokens or dk), and a thread's values are one column's:
// scales are per column, and nothing of one column touches another's.  The
// chain of a chunk is
//   S k^T (MMA) -> R -> T R (MMA) -> d -> d k (MMA) -> S
// with the outputs' products S q^T and d P^T issued behind them.
template <int DK>
struct Stage {
  unsigned char k[C * DK * 2], q[C * DK * 2];
  unsigned char t_hi[kMat], t_lo[kMat], p[kMat];
  unsigned char v[C * kCols * 2];
};

template <int DK>
struct WalkSmem {
  Stage<DK> stage[kStages];
  float f[kStages][kFactors];
  float s_max[2][kCols], r_max[2][kCols];        // [half of dk or of the tokens][column]
  int r_bad[2][kCols];                           // first token whose R is not finite, or C
  float o_s[2][kCols], o_d[2][kCols];            // [buffer][column] factors of S q^T and d P^T
  int o_bad[2][kCols];
  uint64_t full[kStages], empty[kStages];
  uint64_t s_ready, r_ready, d_ready, ks_done, tr_done, u_done, o_done, o_free;
  uint32_t tmem;
};

// TMEM columns.  d's terms replace R's once T R is done; S k^T and T R lie in U's place,
// both read before d k is written there.
constexpr uint32_t kTShi = 0, kTSlo = 64, kTRhi = 128, kTRlo = 160, kTd = 192, kTU = 224, kTKS = 224, kTTR = 288,
                   kTO1 = 352, kTO2 = 416, kTmemCols = 512;

// The wait is bounded; a failure is recorded and the walk goes on with what is there.
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity) {
  if (!mbar_wait(bar, parity)) atomicOr(&g_dn_status, kStatusTimeout);
  __syncwarp();
}

__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

__device__ __forceinline__ void columns_sync() {   // the 8 warps of the recurrence
  __syncwarp();
  asm volatile("bar.sync 1, 256;" ::: "memory");
}

// B operand whose N runs along the rows' bytes (k^T for d k): 64 elements of N per 128-byte row,
// the next 64 C * 128 bytes on, the next 8 of K 1024 bytes on.
__device__ __forceinline__ uint64_t desc_n_major(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | (static_cast<uint64_t>(C * 128 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
constexpr uint32_t kNMajorB = 1u << 16;

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sixteen values of a column, scaled, as the f16 terms of 16 steps of K.
__device__ __forceinline__ void store_terms(const float* v, float s, uint32_t hi_at, uint32_t lo_at) {
  uint32_t hi[8], lo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) split2(v[2 * i] * s, v[2 * i + 1] * s, hi[i], lo[i]);
  tmem_st_x8(hi_at, hi);
  tmem_st_x8(lo_at, lo);
}

// Power-of-two scale for a bound; not finite: the smallest scale.
__device__ __forceinline__ int bound_exp(float bound) {
  return bound < 0x1p127f ? scale_exp(__float_as_uint(bound)) : -112;
}

template <int DK>
__global__ void __launch_bounds__(kThreads, 1) dn_walk_kernel(const DnRows a, const Plan plan, const Work work,
                                                              int64_t slot0, int64_t slot1, bool vec) {
  extern __shared__ unsigned char raw[];
  WalkSmem<DK>& sm = *reinterpret_cast<WalkSmem<DK>*>(raw + ((1024 - (smem_u32(raw) & 1023)) & 1023));
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int cb = (a.dv + kCols - 1) / kCols;
  const int c0 = static_cast<int>(blockIdx.x % cb) * kCols;
  const int h = static_cast<int>(blockIdx.x / cb % a.heads);
  const int64_t seq = blockIdx.x / cb / a.heads;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 33);
      mbar_init(&sm.empty[i], 13);   // 8 + 4 warps, the last MMAs
    }
    mbar_init(&sm.s_ready, 8);
    mbar_init(&sm.r_ready, 8);
    mbar_init(&sm.d_ready, 8);
    mbar_init(&sm.ks_done, 1);
    mbar_init(&sm.tr_done, 1);
    mbar_init(&sm.u_done, 1);
    mbar_init(&sm.o_done, 1);
    mbar_init(&sm.o_free, 4);
    fence_mbar_init();
  }
  pdl_wait();
  const bool ok = !plan.cu || dn_plan_ok(plan.cu, plan.n_seqs, plan.tokens);
  // this launch's chunks of the sequence
  const int64_t begin = ok ? plan.begin(seq) : 0, base = ok ? plan.slot(seq) : slot0;
  const int64_t len = ok ? plan.end(seq) - begin : 0, chunks = (len + C - 1) / C;
  const int64_t first = max(slot0 - base, static_cast<int64_t>(0)), last = min(slot1 - base, chunks);
  if (base >= slot1 || (first > 0 && first >= last)) return;
  const int n = static_cast<int>(max(last - first, static_cast<int64_t>(0)));
  const float* s_from = first > 0 ? a.s_out : a.s_in;
  if (w == 12) tmem_alloc(&sm.tmem, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sm.tmem;

  if (w < 8) {
    // ---- the recurrence: a thread has a column, half of dk and half of a chunk's tokens
    constexpr int NS = DK / 2;
    const int half = w >> 2, L = (w & 3) * 32 + lane, col = c0 + L;
    const bool in = col < a.dv;
    const uint32_t tl = tm + (static_cast<uint32_t>((w & 3) * 32) << 16);
    const int64_t s_at = ((seq * a.heads + h) * DK + half * NS) * static_cast<int64_t>(a.dv) + col;
    float S[NS], inv = 1.f, s_max = 0.f;   // S 2^e; 2^-e; the largest of this half
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      S[i] = in && s_from ? s_from[s_at + i * static_cast<int64_t>(a.dv)] : 0.f;
      s_max = fmaxf(s_max, __uint_as_float(finite_bits(S[i])));
    }
    if (!ok) {
#pragma unroll
      for (int i = 0; i < NS; ++i) S[i] = CUDART_NAN_F;
    }
    if (n > 0) {
      sm.s_max[half][L] = s_max;
      columns_sync();
      const int e = scale_exp(__float_as_uint(fmaxf(s_max, sm.s_max[half ^ 1][L])));
      const float s = exp2i(e);
      inv = exp2i(-e);
#pragma unroll
      for (int i = 0; i < NS; ++i) S[i] *= s;
#pragma unroll
      for (int i = 0; i < NS; i += 16)
        store_terms(&S[i], 1.f, tl + kTShi + (half * NS + i) / 2, tl + kTSlo + (half * NS + i) / 2);
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&sm.s_ready);
    }
    for (int it = 0; it < n; ++it) {
      const uint32_t ph = it & 1, st = it % kStages;
      const float* f = sm.f[st];
      wait(&sm.full[st], (it / kStages) & 1);
      // R = beta v - beta e^G S^T k of 32 tokens
      float R[32];
      {
        uint32_t v[16];   // the column's values of v, two tokens a word
        const uint16_t* vs = reinterpret_cast<const uint16_t*>(sm.stage[st].v) + half * 32 * kCols + L;
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = vs[2 * i * kCols] | static_cast<uint32_t>(vs[(2 * i + 1) * kCols]) << 16;
        wait(&sm.ks_done, ph);
        tc_fence_after();
        uint32_t ks[32];
        tmem_ld_x32(tl + kTKS + half * 32, ks);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 fa = *reinterpret_cast<const float4*>(f + kFA + half * 32 + i);
          const float4 fb = *reinterpret_cast<const float4*>(f + kFB + half * 32 + i);
          R[i] = fmaf(fa.x, __uint_as_float(ks[i]) * inv, fb.x * __uint_as_float(v[i / 2] << 16));
          R[i + 1] = fmaf(fa.y, __uint_as_float(ks[i + 1]) * inv, fb.y * __uint_as_float(v[i / 2] & 0xffff0000u));
          R[i + 2] = fmaf(fa.z, __uint_as_float(ks[i + 2]) * inv, fb.z * __uint_as_float(v[i / 2 + 1] << 16));
          R[i + 3] = fmaf(fa.w, __uint_as_float(ks[i + 3]) * inv, fb.w * __uint_as_float(v[i / 2 + 1] & 0xffff0000u));
        }
      }
      float m4[4] = {};
#pragma unroll
      for (int i = 0; i < 32; ++i) m4[i & 3] = max_nan(m4[i & 3], fabsf(R[i]));
      float m = max_nan(max_nan(m4[0], m4[1]), max_nan(m4[2], m4[3]));
      int bad = C;
      if (!(m < CUDART_INF_F)) {
        // A token's infinity or NaN may not reach the tokens before it through T's and P's zeros:
        // it is taken out here and put back into d from that token on.
        m = 0.f;
#pragma unroll
        for (int i = 31; i >= 0; --i) {
          if (!(fabsf(R[i]) < CUDART_INF_F)) {
            bad = half * 32 + i;
            R[i] = 0.f;
          }
          m = fmaxf(m, fabsf(R[i]));
        }
      }
      sm.r_max[half][L] = m;
      sm.r_bad[half][L] = bad;
      sm.s_max[half][L] = s_max;
      columns_sync();
      m = fmaxf(m, sm.r_max[half ^ 1][L]);
      bad = min(bad, sm.r_bad[half ^ 1][L]);
      const float s_all = fmaxf(s_max, sm.s_max[half ^ 1][L]);
      const int re = scale_exp(__float_as_uint(m));
      {
        const float s = exp2i(re);
#pragma unroll
        for (int i = 0; i < 32; i += 16)
          store_terms(&R[i], s, tl + kTRhi + half * 16 + i / 2, tl + kTRlo + half * 16 + i / 2);
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&sm.r_ready);
      // d = T R.  Its scales come from bounds: R's largest times T's row sums, weighted and not.
      const float4 fe = *reinterpret_cast<const float4*>(f + kFEnd);
      const float w_bound = m * fe.w;
      const int we = bound_exp(w_bound), de = bound_exp(m * f[kFEnd + 4]);
      const float d_inv = w_bound > 0.f ? exp2i(-we) : 0.f;
      {
        const float c1 = exp2i(-re) * fe.y, c16 = c1 * exp2i(de), ws = exp2i(we);
        wait(&sm.tr_done, ph);
        tc_fence_after();
        uint32_t d[32];
        tmem_ld_x32(tl + kTTR + half * 32, d);
#pragma unroll
        for (int i = 0; i < 32; i += 16) {
          uint32_t o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float x = __uint_as_float(d[i + 2 * j]) * c16, y = __uint_as_float(d[i + 2 * j + 1]) * c16;
            if (half * 32 + i + 2 * j >= bad) x = 0.f;
            if (half * 32 + i + 2 * j + 1 >= bad) y = 0.f;
            o[j] = pack_h2(x, y);
          }
          tmem_st_x8(tl + kTd + half * 16 + i / 2, o);
        }
        const float cw = c1 * ws;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 fw = *reinterpret_cast<const float4*>(f + kFW + half * 32 + i);
          R[i] = __uint_as_float(d[i]) * cw * fw.x;
          R[i + 1] = __uint_as_float(d[i + 1]) * cw * fw.y;
          R[i + 2] = __uint_as_float(d[i + 2]) * cw * fw.z;
          R[i + 3] = __uint_as_float(d[i + 3]) * cw * fw.w;
        }
        if (bad < C) R[0] = CUDART_NAN_F;   // the state's column is lost with it
#pragma unroll
        for (int i = 0; i < 32; i += 16)
          store_terms(&R[i], 1.f, tl + kTRhi + half * 16 + i / 2, tl + kTRlo + half * 16 + i / 2);
      }
      if (half == 0) {
        sm.o_s[ph][L] = inv;
        sm.o_d[ph][L] = exp2i(-de) * fe.z;
        sm.o_bad[ph][L] = bad;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.d_ready);
        mbar_arrive(&sm.empty[st]);
      }
      // S = e^G64 S + d k.  Its scale comes from a bound: 64 products of d and k, both below 2^15 as f16.
      const int e = bound_exp(fmaf(s_all, fe.x, d_inv * 0x1p36f));
      const float s = exp2i(e), keep = fe.x * inv * s, gain = d_inv * s;
      inv = exp2i(-e);
      wait(&sm.u_done, ph);
      tc_fence_after();
      float sm4[4] = {};
#pragma unroll
      for (int i = 0; i < NS; i += 16) {
        uint32_t u[16];
        tmem_ld_x16(tl + kTU + half * NS + i, u);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          S[i + j] = fmaf(__uint_as_float(u[j]), gain, S[i + j] * keep);
          sm4[j & 3] = fmaxf(sm4[j & 3], fabsf(S[i + j]));
        }
        store_terms(&S[i], 1.f, tl + kTShi + (half * NS + i) / 2, tl + kTSlo + (half * NS + i) / 2);
      }
      s_max = fmaxf(fmaxf(sm4[0], sm4[1]), fmaxf(sm4[2], sm4[3])) * inv;
      if (!(s_max < CUDART_INF_F)) s_max = 0.f;   // the column is lost; its scale no longer matters
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&sm.s_ready);
    }
    if (in) {
#pragma unroll
      for (int i = 0; i < NS; ++i) a.s_out[s_at + i * static_cast<int64_t>(a.dv)] = S[i] * inv;
    }
  } else if (w < 12) {
    // ---- the outputs: a thread has a column
    const int L = (w & 3) * 32 + lane, col = c0 + L;
    const uint32_t tl = tm + (static_cast<uint32_t>((w & 3) * 32) << 16);
    for (int it = 0; it < n; ++it) {
      const uint32_t ph = it & 1, st = it % kStages;
      const float* f = sm.f[st];
      const int64_t t0 = begin + (first + it) * C;
      const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
      wait(&sm.full[st], (it / kStages) & 1);
      wait(&sm.d_ready, ph);   // for o_s, o_d and o_bad
      wait(&sm.o_done, ph);
      tc_fence_after();
      const float os = sm.o_s[ph][L], od = sm.o_d[ph][L];
      const int bad = sm.o_bad[ph][L];
      uint16_t* dst = a.out + (t0 * a.heads + h) * a.dv + col;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t x[32], y[32];
        tmem_ld_x32(tl + kTO1 + hf * 32, x);
        tmem_ld_x32(tl + kTO2 + hf * 32, y);
        if (hf) {
          tc_fence_before();
          warp_arrive(&sm.o_free);
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 fq = *reinterpret_cast<const float4*>(f + kFQ + hf * 32 + i);
          const float q4[4] = {fq.x, fq.y, fq.z, fq.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int tok = hf * 32 + i + j;
            float o = fmaf(__uint_as_float(y[i + j]), od, __uint_as_float(x[i + j]) * os * q4[j]);
            if (tok >= bad) o = CUDART_NAN_F;
            if (tok < cnt && col < a.dv) dst[static_cast<int64_t>(tok) * a.heads * a.dv] = dn_bf16_bits(o);
          }
        }
      }
      warp_arrive(&sm.empty[st]);
    }
  } else if (w == 12) {
    // ---- the MMAs
    constexpr uint32_t id = idesc_f16(128, C), id_u = idesc_f16(128, DK) | kNMajorB;
    const uint32_t issue = elect_one();
    auto tile = [](uint32_t addr, int kt) { return umma_desc_sw128(addr + (kt >> 2) * (C * 128) + (kt & 3) * 32, 1024); };
    for (int it = 0; it < n; ++it) {
      const uint32_t ph = it & 1, st = it % kStages;
      const Stage<DK>& sg = sm.stage[st];
      const uint32_t k = smem_u32(sg.k), q = smem_u32(sg.q), th = smem_u32(sg.t_hi), tlo = smem_u32(sg.t_lo),
                     p = smem_u32(sg.p);
      wait(&sm.full[st], (it / kStages) & 1);
      wait(&sm.s_ready, ph);
      tc_fence_after();
      if (issue) {
#pragma unroll
        for (int kt = 0; kt < DK / 16; ++kt) {
          mma_f16_ta(tm + kTKS, tm + kTShi + kt * 8, tile(k, kt), id, kt > 0);
          mma_f16_ta(tm + kTKS, tm + kTSlo + kt * 8, tile(k, kt), id, true);
        }
        mma_commit(&sm.ks_done);
      }
      __syncwarp();
      if (it > 0) wait(&sm.o_free, ph ^ 1);
      tc_fence_after();
      if (issue) {
#pragma unroll
        for (int kt = 0; kt < DK / 16; ++kt) mma_f16_ta(tm + kTO1, tm + kTShi + kt * 8, tile(q, kt), id, kt > 0);
      }
      __syncwarp();
      wait(&sm.r_ready, ph);
      tc_fence_after();
      if (issue) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
          mma_f16_ta(tm + kTTR, tm + kTRhi + kt * 8, tile(th, kt), id, kt > 0);
          mma_f16_ta(tm + kTTR, tm + kTRlo + kt * 8, tile(th, kt), id, true);
          mma_f16_ta(tm + kTTR, tm + kTRhi + kt * 8, tile(tlo, kt), id, true);
        }
        mma_commit(&sm.tr_done);
      }
      __syncwarp();
      wait(&sm.d_ready, ph);
      tc_fence_after();
      if (issue) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
          const uint64_t b = desc_n_major(k + kt * 2048);
          mma_f16_ta(tm + kTU, tm + kTRhi + kt * 8, b, id_u, kt > 0);
          mma_f16_ta(tm + kTU, tm + kTRlo + kt * 8, b, id_u, true);
        }
        mma_commit(&sm.u_done);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) mma_f16_ta(tm + kTO2, tm + kTd + kt * 8, tile(p, kt), id, kt > 0);
        mma_commit(&sm.o_done);
        mma_commit(&sm.empty[st]);
      }
      __syncwarp();
    }
  } else {
    // ---- the copies
    asm volatile("fence.proxy.async.global;" ::: "memory");   // the other kernel's stores, before bulk copies of them
    const int key_heads = a.heads / a.ratio;
    for (int it = 0; it < n; ++it) {
      const uint32_t st = it % kStages;
      Stage<DK>& sg = sm.stage[st];
      const int64_t ci = first + it, t0 = begin + ci * C, slot = base + ci - slot0;
      const int cnt = static_cast<int>(min(static_cast<int64_t>(C), begin + len - t0));
      const unsigned char* kq = work.kq + (slot * key_heads + h / a.ratio) * (2 * C * DK * 2);
      const unsigned char* head = work.heads + (slot * a.heads + h) * static_cast<int64_t>(kHeadBytes);
      if (it >= kStages) wait(&sm.empty[st], (it / kStages + 1) & 1);
      if (lane == 0) {
        mbar_arrive_expect_tx(&sm.full[st], 2 * C * DK * 2 + kHeadBytes);
        bulk_g2s(sg.k, kq, 2 * C * DK * 2, &sm.full[st]);
        bulk_g2s(sg.t_hi, head, 2 * kMat, &sm.full[st]);
        bulk_g2s(sm.f[st], head + 2 * kMat, kFactors * 4, &sm.full[st]);
        bulk_g2s(sg.p, head + kRecBytes, kMat, &sm.full[st]);
      }
      __syncwarp();
      const uint16_t* v = a.v + t0 * a.v_row + h * a.v_head + c0;
      const int ch = lane & 15, cols = min(a.dv - c0, kCols);
      const bool in = ch * 8 < cols;
#pragma unroll 8
      for (int i = 0; i < C / 2; ++i) {
        const int r = i * 2 + (lane >> 4);
        const uint32_t dst = smem_u32(sg.v) + r * (kCols * 2) + ch * 16;
        const bool live = in && r < cnt;
        const uint16_t* src = v + (live ? r * a.v_row + ch * 8 : 0);
        if (vec) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
        } else {
          uint32_t x[4] = {0, 0, 0, 0};
          if (live)
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
    }
    // nothing of this warp may still be on its way when the block ends
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (w == 12) tmem_dealloc(tm, kTmemCols);
}

}  // namespace

// ------------------------------------------------------------------ host
namespace {

// Chunks are taken in segments whose workspace stays within this, so that
// what dn_prep_kernel writes is still in L2 when dn_walk_kernel reads it.
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
  const int64_t blocks = n_seqs * a.heads * ((a.dv + kCols - 1) / kCols);
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
    e = cudaFuncSetAttribute(dn_walk_kernel<DK>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(WalkSmem<DK>) + 1024);
  if (e != cudaSuccess) return set_error(QFN_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
  const Plan plan{cu, n_seqs, tokens};
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const Work work{ws, ws + seg * key_heads * (2 * C * DK * 2)};
  for (int64_t s0 = 0; s0 < slots && e == cudaSuccess; s0 += seg) {
    const int64_t s1 = s0 + seg < slots ? s0 + seg : slots;
    e = launch(dn_prep_kernel<DK>, (s1 - s0) * key_heads, kPrepThreads, sizeof(PrepSmem<DK>), as_stream(stream), a, plan,
               work, s0, kq_vec);
    if (e == cudaSuccess)
      e = launch(dn_walk_kernel<DK>, blocks, kThreads, sizeof(WalkSmem<DK>) + 1024, as_stream(stream), a, plan, work, s0, s1,
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
