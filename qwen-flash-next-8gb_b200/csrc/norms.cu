// The norms of a layer around its blocks (RMSNorm in fp32, one rounding per
// output):
//
//   qfn_gated_norm     y = x * rsqrt(mean x^2 + eps) * w * silu(z), per head
//   qfn_norm_residual  p  = block * rsqrt(mean block^2 + eps) * w_post
//                      r' = residual + scale * gate * p
//                      n  = r' * rsqrt(mean r'^2 + eps) * w_next
//
// Both are bound by memory: a row is read once, held in registers as fp32
// through its sums, and written once.  n is formed from r' before its
// rounding, so each output carries one rounding.  Rows whose bases, strides and length allow it move
// in 16-byte pieces of 8 elements (two for fp32); the others go by two elements or one.
#include <cuda_bf16.h>

#include "common.cuh"
#include "host.cuh"

namespace qfn {

// Element types of one operand.
__device__ __forceinline__ float load1(const void* p, int dtype, int64_t i) {
  return dtype == QFN_DTYPE_F32 ? static_cast<const float*>(p)[i]
                                : bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ void store1(void* p, int dtype, int64_t i, float v) {
  if (dtype == QFN_DTYPE_F32) {
    static_cast<float*>(p)[i] = v;
  } else {
    const __nv_bfloat16 b = __float2bfloat16_rn(v);
    static_cast<uint16_t*>(p)[i] = *reinterpret_cast<const uint16_t*>(&b);
  }
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// Eight neighbouring elements, 16-byte aligned (32 bytes for fp32).
__device__ __forceinline__ void unpack8(uint4 u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const void* p, int dtype, int64_t i, float (&v)[8]) {
  if (dtype == QFN_DTYPE_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    unpack8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i), v);
  }
}
__device__ __forceinline__ void store8(void* p, int dtype, int64_t i, const float (&v)[8]) {
  if (dtype == QFN_DTYPE_F32) {
    float* f = static_cast<float*>(p) + i;
    *reinterpret_cast<float4*>(f) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(f + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
  }
}

// 1 / (1 + e^-x) from the special-function unit's exp2 and reciprocal, as 2^-24 / (2^-24 + 2^-24 e^-x): so neither the
// exponential nor the reciprocal leaves fp32's normal numbers before the result is below 2^-149 (silu(-89) = -2e-37 is
// a normal number although sigmoid(-89) is none).  The two are each within 2 steps of fp32; the rounding of
// x log2(e) + 24 moves the exponential by 2^-20 at most around zero, by |x| 2^-23 far from it.  (With expf and a true
// division the gated norm was bound by its instructions: 106 us for 16384 x 32 rows of 128.)
__device__ __forceinline__ float sigmoidf(float x) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(x, -1.44269504f, -24.f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(0x1p-24f + e));
  return r * 0x1p-24f;
}

// ------------------------------------------------------------------ gated norm
struct GatedNorm {
  const uint16_t *x, *z;
  const void* w;
  uint16_t* y;   // [rows][heads][dim], contiguous
  int64_t x_row, x_head, z_row, z_head, n;   // n = rows * heads
  int w_dtype, heads, dim;
  float eps;
};

// LANES lanes of a warp share one row of dim <= 8 LANES; a thread takes its
// piece of ROWS rows, one block's worth apart, and requests all of them first.
// Measured: 16384 x 32 rows of 128 in 69 to 76 us, 5.3 to 5.8 TB/s (issue slots 70 %).
template <int LANES, int ROWS>
__global__ void __launch_bounds__(256) gated_norm_kernel(const GatedNorm a) {
  constexpr int kPer = 256 / LANES;   // rows of a block at a time
  pdl_wait();
  pdl_launch_dependents();
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (kPer * ROWS) + threadIdx.x / LANES;   // n < 2^31
  const int c = static_cast<int>(threadIdx.x % LANES) * 8;
  const bool col = c < a.dim;
  uint4 xr[ROWS], zr[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int64_t i = i0 + k * kPer;
    const uint32_t row = static_cast<uint32_t>(i) / static_cast<uint32_t>(a.heads),
                   h = static_cast<uint32_t>(i) - row * static_cast<uint32_t>(a.heads);
    xr[k] = zr[k] = make_uint4(0, 0, 0, 0);
    if (col && i < a.n) {
      xr[k] = *reinterpret_cast<const uint4*>(a.x + row * a.x_row + h * a.x_head + c);
      zr[k] = *reinterpret_cast<const uint4*>(a.z + row * a.z_row + h * a.z_head + c);
    }
  }
  float w[8] = {};
  if (col) load8(a.w, a.w_dtype, c, w);
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int64_t i = i0 + k * kPer;
    float x[8], z[8], ss = 0.f;
    unpack8(xr[k], x);
    unpack8(zr[k], z);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!col || i >= a.n) continue;
    const float r = rsqrtf(ss / static_cast<float>(a.dim) + a.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] * r * w[j] * (z[j] * sigmoidf(z[j]));
    store8(a.y, QFN_DTYPE_BF16, i * a.dim + c, x);
  }
}

// Any dim and alignment: a warp per row, read twice (the second time from L1).
__global__ void __launch_bounds__(256) gated_norm_any_kernel(const GatedNorm a) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  if (i >= a.n) return;
  const int lane = threadIdx.x & 31;
  const uint16_t* x = a.x + i / a.heads * a.x_row + i % a.heads * a.x_head;
  const uint16_t* z = a.z + i / a.heads * a.z_row + i % a.heads * a.z_head;
  float ss = 0.f;
  for (int c = lane; c < a.dim; c += 32) {
    const float v = bf16_bits_to_f32(x[c]);
    ss = fmaf(v, v, ss);
  }
  const float r = rsqrtf(warp_sum(ss) / static_cast<float>(a.dim) + a.eps);
  for (int c = lane; c < a.dim; c += 32) {
    const float g = bf16_bits_to_f32(z[c]);
    store1(a.y, QFN_DTYPE_BF16, i * a.dim + c, bf16_bits_to_f32(x[c]) * r * load1(a.w, a.w_dtype, c) * (g * sigmoidf(g)));
  }
}

// ------------------------------------------------------------------ norm, gate, residual, norm
struct NormResidual {
  const void *block, *residual, *w_post, *gate, *w_next;
  void* r_out;
  uint16_t* n_out;
  int64_t block_row, residual_row, gate_row;
  int block_dtype, residual_dtype, post_dtype, gate_dtype, next_dtype;
  int gate_kind;   // 0 none, 1 a value per row, 2 a value per element
  int sigmoid, dim;
  float scale, eps;
};

// Sum over the block of up to 32 warps; every thread gets it.  red: 33 floats.
__device__ __forceinline__ float block_sum(float v, float* red) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  v = warp_sum(v);
  if (lane == 0) red[w] = v;
  __syncthreads();
  float t = lane < nw ? red[lane] : 0.f;
  return warp_sum(t);
}

// Rows of one 8-element piece a thread (dim <= 8 x 512).  A CTA takes row after
// row, gridDim.x apart, and requests the next row's block, residual and gate
// while this one's sums are formed, so that two barriers a row leave no gap
// in the stream of loads.  F32 flags: the operands' types; read at run time they
// spilled registers (184 us).  Measured: 16384 rows of 2560 bf16 in 77 to 83 us,
// 5.1 to 5.4 TB/s.
constexpr int kPieceThreads = 512;

template <bool F32>
struct Piece {
  uint4 u[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    const uint4* q = F32 ? reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i)
                         : reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    u[0] = q[0];
    if (F32) u[F32 ? 1 : 0] = q[F32 ? 1 : 0];
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if (F32) {
      const uint4 b = u[F32 ? 1 : 0];
      const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    } else {
      unpack8(u[0], v);
    }
  }
};

template <bool BF, bool RF, bool GF>
__global__ void __launch_bounds__(kPieceThreads, 2) norm_residual_piece_kernel(const NormResidual a, int64_t rows) {
  __shared__ float red[2][2][32];   // [row parity]: a slow warp may still read the last row's sums
  pdl_wait();
  pdl_launch_dependents();
  const int c = threadIdx.x * 8;
  const bool in = c < a.dim, per_element = a.gate_kind == 2;
  Piece<BF> bp;
  Piece<RF> rp;
  Piece<GF> gp;
  auto request = [&](int64_t row) {
    if (row >= rows || !in) return;
    bp.load(a.block, row * a.block_row + c);
    rp.load(a.residual, row * a.residual_row + c);
    if (per_element) gp.load(a.gate, row * a.gate_row + c);
  };
  request(blockIdx.x);
  int parity = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, parity ^= 1) {
    float b[8] = {}, v[8] = {}, ss = 0.f;
    if (in) bp.get(b);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(b[j], b[j], ss);
    if (in && per_element) {   // the gated block; the norm's factor comes later
      gp.get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] *= a.sigmoid ? sigmoidf(v[j]) : v[j];
    }
    if (in) rp.get(v);
    request(row + gridDim.x);
    float m = a.scale;
    if (a.gate_kind == 1) {
      const float g = load1(a.gate, a.gate_dtype, row * a.gate_row);
      m *= a.sigmoid ? sigmoidf(g) : g;
    }
    if (a.w_post) {
      m *= rsqrtf(block_sum(ss, red[parity][0]) / static_cast<float>(a.dim) + a.eps);
      if (in) {
        float w[8];
        load8(a.w_post, a.post_dtype, c, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] *= w[j];
      }
    }
    float s2 = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = fmaf(b[j], m, v[j]);
      s2 = fmaf(v[j], v[j], s2);
    }
    if (in) store8(a.r_out, RF ? QFN_DTYPE_F32 : QFN_DTYPE_BF16, row * a.dim + c, v);
    if (!a.w_next) continue;
    const float rn = rsqrtf(block_sum(s2, red[parity][1]) / static_cast<float>(a.dim) + a.eps);
    if (in) {
      float w[8];
      load8(a.w_next, a.next_dtype, c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] *= v[j] * rn;
      store8(a.n_out, QFN_DTYPE_BF16, row * a.dim + c, w);
    }
  }
}

// Other rows: CTA = one row; a thread holds PARTS pieces of WIDTH neighbouring
// elements, blockDim.x pieces apart: 8 where 16-byte pieces are possible
// (dim > 4096), 2 or 1 where alignment or dim rule them out.  The type is
// asked once for all of an operand's pieces, so that their loads go out together.
template <int WIDTH, bool F32>
__device__ __forceinline__ void load_piece(const void* p, int64_t i, float (&v)[WIDTH]) {
  if constexpr (WIDTH == 8) {
    load8(p, F32 ? QFN_DTYPE_F32 : QFN_DTYPE_BF16, i, v);
  } else if constexpr (WIDTH == 2) {
    if constexpr (F32) {
      const float2 f = *reinterpret_cast<const float2*>(static_cast<const float*>(p) + i);
      v[0] = f.x;
      v[1] = f.y;
    } else {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i);
      v[0] = __uint_as_float(u << 16);
      v[1] = __uint_as_float(u & 0xffff0000u);
    }
  } else {
    v[0] = load1(p, F32 ? QFN_DTYPE_F32 : QFN_DTYPE_BF16, i);
  }
}
template <int WIDTH, int PARTS, bool F32>
__device__ __forceinline__ void load_row_as(const void* p, int64_t base, int dim, float (&v)[PARTS][WIDTH]) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    const int c = (k * blockDim.x + threadIdx.x) * WIDTH;
#pragma unroll
    for (int j = 0; j < WIDTH; ++j) v[k][j] = 0.f;
    if (c < dim) load_piece<WIDTH, F32>(p, base + c, v[k]);
  }
}
template <int WIDTH, int PARTS>
__device__ __forceinline__ void load_row(const void* p, int dtype, int64_t base, int dim, float (&v)[PARTS][WIDTH]) {
  if (dtype == QFN_DTYPE_F32) load_row_as<WIDTH, PARTS, true>(p, base, dim, v);
  else load_row_as<WIDTH, PARTS, false>(p, base, dim, v);
}
template <int WIDTH, int PARTS, bool F32>
__device__ __forceinline__ void store_row_as(void* p, int64_t base, int dim, const float (&v)[PARTS][WIDTH]) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    const int c = (k * blockDim.x + threadIdx.x) * WIDTH;
    if (c >= dim) continue;
    constexpr int dtype = F32 ? QFN_DTYPE_F32 : QFN_DTYPE_BF16;
    if constexpr (WIDTH == 8) store8(p, dtype, base + c, v[k]);
    else if constexpr (WIDTH == 2 && F32)
      *reinterpret_cast<float2*>(static_cast<float*>(p) + base + c) = make_float2(v[k][0], v[k][1]);
    else if constexpr (WIDTH == 2)
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p) + base + c) = pack2(v[k][0], v[k][1]);
    else store1(p, dtype, base + c, v[k][0]);
  }
}

template <int WIDTH, int PARTS, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_residual_kernel(const NormResidual a) {
  // what is requested before the block's norm is known; the rest comes after it
  constexpr bool kAhead = PARTS * WIDTH <= 16;
  __shared__ float red[2][32];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  float b[PARTS][WIDTH], r[PARTS][WIDTH], g[PARTS][WIDTH], ss = 0.f;
  load_row(a.block, a.block_dtype, row * a.block_row, a.dim, b);
  if constexpr (kAhead) {
    load_row(a.residual, a.residual_dtype, row * a.residual_row, a.dim, r);
    if (a.gate_kind == 2) load_row(a.gate, a.gate_dtype, row * a.gate_row, a.dim, g);
  }
#pragma unroll
  for (int k = 0; k < PARTS; ++k)
#pragma unroll
    for (int j = 0; j < WIDTH; ++j) ss = fmaf(b[k][j], b[k][j], ss);
  float m = a.scale;
  if (a.gate_kind == 1) {
    const float x = load1(a.gate, a.gate_dtype, row * a.gate_row);
    m *= a.sigmoid ? sigmoidf(x) : x;
  }
  if (a.w_post) m *= rsqrtf(block_sum(ss, red[0]) / static_cast<float>(a.dim) + a.eps);
#pragma unroll
  for (int k = 0; k < PARTS; ++k)
#pragma unroll
    for (int j = 0; j < WIDTH; ++j) b[k][j] *= m;
  if (a.gate_kind == 2) {
    if constexpr (!kAhead) load_row(a.gate, a.gate_dtype, row * a.gate_row, a.dim, g);
#pragma unroll
    for (int k = 0; k < PARTS; ++k)
#pragma unroll
      for (int j = 0; j < WIDTH; ++j) b[k][j] *= a.sigmoid ? sigmoidf(g[k][j]) : g[k][j];
  }
  if (a.w_post) {
    load_row(a.w_post, a.post_dtype, 0, a.dim, g);
#pragma unroll
    for (int k = 0; k < PARTS; ++k)
#pragma unroll
      for (int j = 0; j < WIDTH; ++j) b[k][j] *= g[k][j];
  }
  if constexpr (!kAhead) load_row(a.residual, a.residual_dtype, row * a.residual_row, a.dim, r);
  float s2 = 0.f;
#pragma unroll
  for (int k = 0; k < PARTS; ++k)
#pragma unroll
    for (int j = 0; j < WIDTH; ++j) {
      b[k][j] += r[k][j];
      s2 = fmaf(b[k][j], b[k][j], s2);
    }
  if (a.residual_dtype == QFN_DTYPE_F32) store_row_as<WIDTH, PARTS, true>(a.r_out, row * a.dim, a.dim, b);
  else store_row_as<WIDTH, PARTS, false>(a.r_out, row * a.dim, a.dim, b);
  if (!a.w_next) return;
  const float rn = rsqrtf(block_sum(s2, red[1]) / static_cast<float>(a.dim) + a.eps);
  load_row(a.w_next, a.next_dtype, 0, a.dim, g);
#pragma unroll
  for (int k = 0; k < PARTS; ++k)
#pragma unroll
    for (int j = 0; j < WIDTH; ++j) g[k][j] *= b[k][j] * rn;
  store_row_as<WIDTH, PARTS, false>(a.n_out, row * a.dim, a.dim, g);
}

namespace {

template <typename Kernel, typename... Args>
int launch(const char* what, Kernel kernel, int64_t blocks, int threads, qfn_stream_t stream, const Args&... args) {
  QFN_REQUIRE(blocks <= 0x7fffffff, QFN_ERR_UNSUPPORTED, "%s: too many rows", what);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.stream = as_stream(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return set_error(QFN_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

bool dtype_ok(int d) { return d == QFN_DTYPE_F32 || d == QFN_DTYPE_BF16; }

// Whether rows at p, row_a and row_b elements apart, can be moved 8 elements at a time (16 bytes), or two.
bool wide(const void* p, int dtype, int64_t row_a, int64_t row_b) {
  return !p || (aligned(p, 16) && (row_a * (dtype == QFN_DTYPE_F32 ? 4 : 2)) % 16 == 0 &&
                (row_b * (dtype == QFN_DTYPE_F32 ? 4 : 2)) % 16 == 0);
}
bool two(const void* p, int dtype, int64_t row) {
  return !p || (aligned(p, dtype == QFN_DTYPE_F32 ? 8 : 4) && row % 2 == 0);
}

}  // namespace

}  // namespace qfn

using namespace qfn;

extern "C" int qfn_gated_norm(const uint16_t* x, int64_t x_row, int64_t x_head, const uint16_t* z, int64_t z_row,
                              int64_t z_head, const void* w, int w_dtype, uint16_t* y, int64_t rows, int heads,
                              int dim, float eps, qfn_stream_t stream) {
  constexpr const char* what = "qfn_gated_norm";
  QFN_REQUIRE(rows >= 0 && heads >= 1 && dim >= 1, QFN_ERR_INVALID_ARG, "%s: rows=%lld, heads=%d, dim=%d", what,
              static_cast<long long>(rows), heads, dim);
  QFN_REQUIRE(dtype_ok(w_dtype), QFN_ERR_INVALID_ARG, "%s: w_dtype=%d", what, w_dtype);
  if (rows == 0) return QFN_OK;
  QFN_REQUIRE(x && z && w && y, QFN_ERR_INVALID_ARG, "%s: null pointer", what);
  DeviceInfo* dev;
  const int rc = current_device(&dev);
  if (rc) return rc;
  const GatedNorm a{x, z, w, y, x_row, x_head, z_row, z_head, rows * heads, w_dtype, heads, dim, eps};
  const bool v = dim % 8 == 0 && dim <= 256 && a.n < (int64_t{1} << 31) && wide(x, QFN_DTYPE_BF16, x_row, x_head) &&
                 wide(z, QFN_DTYPE_BF16, z_row, z_head) && wide(w, w_dtype, 0, 0) && aligned(y, 16);
  if (!v) return launch(what, gated_norm_any_kernel, (a.n + 7) / 8, 256, stream, a);
  // four rows a thread keep more bytes on their way; below a wave of blocks of them, one row a thread
  const int lanes = dim <= 64 ? 8 : dim <= 128 ? 16 : 32;
  const int rows_of = a.n >= int64_t{4} * (256 / lanes) * dev->sm_count ? 4 : 1;
  auto kernel = rows_of == 4 ? (lanes == 8 ? gated_norm_kernel<8, 4> : lanes == 16 ? gated_norm_kernel<16, 4>
                                                                                : gated_norm_kernel<32, 4>)
                             : (lanes == 8 ? gated_norm_kernel<8, 1> : lanes == 16 ? gated_norm_kernel<16, 1>
                                                                                : gated_norm_kernel<32, 1>);
  const int64_t per = static_cast<int64_t>(256 / lanes) * rows_of;
  return launch(what, kernel, (a.n + per - 1) / per, 256, stream, a);
}

extern "C" int qfn_norm_residual(const void* block, int block_dtype, int64_t block_row, const void* residual,
                                 int residual_dtype, int64_t residual_row, const void* w_post, int post_dtype,
                                 const void* gate, int gate_kind, int gate_dtype, int64_t gate_row, int gate_sigmoid,
                                 float scale, const void* w_next, int next_dtype, void* residual_out,
                                 uint16_t* normed, int64_t rows, int dim, float eps, qfn_stream_t stream) {
  constexpr const char* what = "qfn_norm_residual";
  QFN_REQUIRE(rows >= 0 && dim >= 1, QFN_ERR_INVALID_ARG, "%s: rows=%lld, dim=%d", what, static_cast<long long>(rows),
              dim);
  QFN_REQUIRE(dim <= 32768, QFN_ERR_UNSUPPORTED, "%s: dim=%d (at most 32768)", what, dim);
  QFN_REQUIRE(dtype_ok(block_dtype) && dtype_ok(residual_dtype) && dtype_ok(post_dtype) && dtype_ok(gate_dtype) &&
                  dtype_ok(next_dtype) && gate_kind >= 0 && gate_kind <= 2,
              QFN_ERR_INVALID_ARG, "%s: unknown dtype or gate kind", what);
  if (rows == 0) return QFN_OK;
  QFN_REQUIRE(block && residual && residual_out && (gate || !gate_kind) && (normed || !w_next), QFN_ERR_INVALID_ARG,
              "%s: null pointer", what);
  DeviceInfo* dev;
  const int rc = current_device(&dev);
  if (rc) return rc;
  const NormResidual a{block, residual, w_post, gate, w_next, residual_out, normed, block_row, residual_row, gate_row,
                       block_dtype, residual_dtype, post_dtype, gate_dtype, next_dtype, gate_kind, gate_sigmoid, dim,
                       scale, eps};
  const bool v = dim % 8 == 0 && wide(block, block_dtype, block_row, 0) &&
                 wide(residual, residual_dtype, residual_row, 0) && wide(w_post, post_dtype, 0, 0) &&
                 (gate_kind != 2 || wide(gate, gate_dtype, gate_row, 0)) && wide(w_next, next_dtype, 0, 0) &&
                 aligned(residual_out, 16) && aligned(normed, 16);
  const int pieces = v ? dim / 8 : dim;
  if (v && pieces <= kPieceThreads) {
    const int threads = (pieces + 31) / 32 * 32;
    const bool bf = block_dtype == QFN_DTYPE_F32, rf = residual_dtype == QFN_DTYPE_F32, gf = gate_dtype == QFN_DTYPE_F32;
    auto kernel = bf ? (rf ? (gf ? norm_residual_piece_kernel<true, true, true> : norm_residual_piece_kernel<true, true, false>)
                           : (gf ? norm_residual_piece_kernel<true, false, true> : norm_residual_piece_kernel<true, false, false>))
                     : (rf ? (gf ? norm_residual_piece_kernel<false, true, true> : norm_residual_piece_kernel<false, true, false>)
                           : (gf ? norm_residual_piece_kernel<false, false, true> : norm_residual_piece_kernel<false, false, false>));
    // as many CTAs as are resident at 64 registers a thread
    const int64_t resident = static_cast<int64_t>(dev->sm_count) * (1024 / threads);
    return launch(what, kernel, rows < resident ? rows : resident, threads, stream, a, rows);
  }
  if (v) {
    const int parts = (pieces + 1023) / 1024, per = (pieces + parts - 1) / parts;
    auto kernel = parts <= 1 ? norm_residual_kernel<8, 1, 1024>
                             : parts <= 2 ? norm_residual_kernel<8, 2, 1024> : norm_residual_kernel<8, 4, 1024>;
    return launch(what, kernel, rows, (per + 31) / 32 * 32, stream, a);
  }
  const bool pairs = dim % 2 == 0 && two(block, block_dtype, block_row) && two(residual, residual_dtype, residual_row) &&
                     two(w_post, post_dtype, 0) && (gate_kind != 2 || two(gate, gate_dtype, gate_row)) &&
                     two(w_next, next_dtype, 0) && two(residual_out, residual_dtype, 0) && two(normed, QFN_DTYPE_BF16, 0);
  const int n = pairs ? dim / 2 : dim;
  // up to 512 threads with all of a row's pieces on their way at once; longer rows, 1024 threads in two steps
  if (n <= 4096) {
    const int parts = n <= 512 ? 2 : n <= 2048 ? 4 : 8;
    const int threads = ((n + parts - 1) / parts + 31) / 32 * 32;
    auto kernel = pairs ? (parts == 2 ? norm_residual_kernel<2, 2, 512> : parts == 4 ? norm_residual_kernel<2, 4, 512>
                                                                                     : norm_residual_kernel<2, 8, 512>)
                        : (parts == 2 ? norm_residual_kernel<1, 2, 512> : parts == 4 ? norm_residual_kernel<1, 4, 512>
                                                                                     : norm_residual_kernel<1, 8, 512>);
    return launch(what, kernel, rows, threads, stream, a);
  }
  const int parts1 = (dim + 1023) / 1024, threads = ((dim + parts1 - 1) / parts1 + 31) / 32 * 32;
  auto kernel = parts1 <= 8 ? norm_residual_kernel<1, 8, 1024> : norm_residual_kernel<1, 32, 1024>;
  return launch(what, kernel, rows, threads, stream, a);
}
