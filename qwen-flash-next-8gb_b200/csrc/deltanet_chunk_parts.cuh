// What the kernels of deltanet_chunk.cu share: the workspace's layout, bf16
// terms, fragments, the sequences' plan.
#pragma once

#include "deltanet_batch.cuh"

namespace qfn {
namespace {

constexpr int C = 64;            // tokens of a chunk
constexpr int kSorted = 64;      // sequences up to which the longest are walked first
constexpr int kPrepThreads = 256;
constexpr int kGS = 68;          // row pitch of the 64 x 64 fp32 matrices of dn_prep_kernel

// Lower triangular 64 x 64 matrices (T, P) are kept as their 10 blocks of 16 x 16
// on and below the diagonal, each term by itself: a block is its four 8 x 8
// quarters, rows of 16 bytes, so that a warp's ldmatrix of a block reads 512
// bytes in the lanes' order.
constexpr int kBlockBytes = 512, kTermBytes = 10 * kBlockBytes;
__host__ __device__ constexpr int tri_block(int i, int j) { return (i * (i + 1) / 2 + j) * kBlockBytes; }
__device__ __forceinline__ uint32_t tri_at(int row, int col8) {   // the 16 bytes of row `row`, columns 8 col8 .. + 7
  return tri_block(row >> 4, col8 >> 1) + ((row >> 3 & 1) * 2 + (col8 & 1)) * 128 + (row & 7) * 16;
}

// Per chunk and value head: T in three terms, the tokens' factors and e^G64, then P in two terms.
enum { kFA = 0, kFB = C, kFQ = 2 * C, kFW = 3 * C, kFEnd = 4 * C };   // -beta e^G ck, beta, e^G cq, e^(G64 - G) ck; e^G64
constexpr int kFactors = 4 * C + 4;
constexpr int kRecBytes = 3 * kTermBytes + kFactors * 4;
constexpr int kPBytes = 2 * kTermBytes;
constexpr int kHeadBytes = kRecBytes + kPBytes;

__device__ unsigned int g_dn_status;

struct Work {
  unsigned char* kq;     // [slots][key heads][2][64][dk] bf16
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

__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// Two values less their bf16 roundings in u, exactly.
__device__ __forceinline__ void less(float& a, float& b, uint32_t u) {
  a -= __uint_as_float(u << 16);
  b -= __uint_as_float(u & 0xffff0000u);
}

// Two values as sums of bf16 terms.  Three terms hold fp32's 24 bits: 8 each, and what two leave has no more
// than 8 bits, so that its upper half is all of it.  A term has fp32's exponent, so no value needs a scale, and
// none loses digits to a larger one beside it.  Two terms are within 2^-16.
__device__ __forceinline__ void split(float a, float b, uint32_t (&u)[3]) {
  u[0] = pack_bf2(a, b);
  less(a, b, u[0]);
  u[1] = pack_bf2(a, b);
  less(a, b, u[1]);
  u[2] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
}
__device__ __forceinline__ void split(float a, float b, uint32_t (&u)[2]) {
  u[0] = pack_bf2(a, b);
  less(a, b, u[0]);
  u[1] = pack_bf2(a, b);
}

// max(m, |a|, |b|), NaN kept
__device__ __forceinline__ float max_abs_nan(float m, float a, float b) {
  asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(a), "f"(b));
  return m;
}

// D += A B and, for the first product of an accumulator, D = A B.  Not volatile: the compiler may
// move the products between the loads.
__device__ __forceinline__ void mma_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
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

// Whether any of a warp's values is not finite.
template <int N>
__device__ __forceinline__ bool any_not_finite(const float (&v)[N][4]) {
  float m0 = 0.f, m1 = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m0 = max_abs_nan(m0, v[i][0], v[i][1]);
    m1 = max_abs_nan(m1, v[i][2], v[i][3]);
  }
  return __any_sync(0xffffffffu, !(max_abs_nan(m0, m1, 0.f) < CUDART_INF_F));
}

// Accumulators of two neighbouring 16 x 8 tiles as the fragments of a 16 x 16 operand's N terms.
template <int N>
__device__ __forceinline__ void frag_split(const float (&a)[4], const float (&b)[4], uint32_t (&f)[N][4]) {
  const float v[4][2] = {{a[0], a[1]}, {a[2], a[3]}, {b[0], b[1]}, {b[2], b[3]}};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t u[N];
    split(v[i][0], v[i][1], u);
#pragma unroll
    for (int n = 0; n < N; ++n) f[n][i] = u[n];
  }
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
