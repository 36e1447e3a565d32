// What the kernels of deltanet_chunk.cu share: the workspace's layout, scales
// and f16 terms, fragments, the sequences' plan.
#pragma once

#include "deltanet_batch.cuh"

namespace qfn {
namespace {

constexpr int C = 64;            // tokens of a chunk
constexpr int kSorted = 64;      // sequences up to which the longest are walked first
constexpr int kPrepThreads = 256;
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
  int64_t n_seqs, tokens, each;   // each: without cu, tokens / n_seqs (a 64-bit division takes a block hundreds of cycles)
  __device__ int64_t begin(int64_t n) const { return cu ? cu[n] : n * each; }
  __device__ int64_t end(int64_t n) const { return cu ? cu[n + 1] : (n + 1) * each; }
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

// The wait is bounded; a failure is recorded and the walk goes on with what is there.
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity) {
  if (!mbar_wait(bar, parity)) atomicOr(&g_dn_status, kStatusTimeout);
  __syncwarp();
}

// max(m, magnitudes of a lane's values), NaN dropped.
template <int N>
__device__ __forceinline__ float lane_max(const float (&v)[N][4]) {
  float m0 = 0.f, m1 = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m0 = max_abs(m0, v[i][0], v[i][1]);
    m1 = max_abs(m1, v[i][2], v[i][3]);
  }
  return fmaxf(m0, m1);
}

// The largest finite magnitude of a warp's values, the same in every lane.
template <int N>
__device__ __forceinline__ float warp_max(const float (&v)[N][4]) {
  uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(lane_max(v)));
  if (b >= 0x7f800000u) {   // an infinity somewhere: the other columns keep their scale
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

// A block's part of a launch: chunks first .. last - 1 of a sequence.
struct Part {
  int64_t seq, begin, len, base;   // the sequence, its first token and tokens, its first slot
  int64_t first, last;
  bool ok;                         // the sequence bounds rise
  __device__ __forceinline__ bool none(int64_t slot1) const { return base >= slot1 || (first > 0 && first >= last); }
};

// Blocks start in order and a sequence's walk cannot be split, so the longest go first: block n takes the
// sequence with n longer ones (equal ones in their order).  Worth its n_seqs^2 steps for few sequences only.
// Ends with the block in step.
__device__ __forceinline__ Part choose(const Plan& plan, int64_t seq, int64_t slot0, int64_t slot1, int* length, int* chosen) {
  Part p;
  p.ok = !plan.cu || dn_plan_ok(plan.cu, plan.n_seqs, plan.tokens);
  if (p.ok && plan.cu && plan.n_seqs <= kSorted) {
    const int n = static_cast<int>(plan.n_seqs), i = threadIdx.x;   // blocks have more threads than kSorted
    if (i < n) length[i] = plan.cu[i + 1] - plan.cu[i];
    __syncthreads();
    if (i < n) {
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += length[j] > length[i] || (length[j] == length[i] && j < i);
      if (rank == seq) *chosen = i;
    }
    __syncthreads();
    seq = *chosen;
  }
  __syncthreads();
  p.seq = seq;
  p.begin = p.ok ? plan.begin(seq) : 0;
  p.base = p.ok ? plan.slot(seq) : slot0;
  p.len = p.ok ? plan.end(seq) - p.begin : 0;
  p.first = max(slot0 - p.base, static_cast<int64_t>(0));
  p.last = min(slot1 - p.base, (p.len + C - 1) / C);
  return p;
}

}  // namespace
}  // namespace qfn
