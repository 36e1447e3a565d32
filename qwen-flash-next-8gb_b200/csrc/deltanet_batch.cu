// The gated delta rule (qwen_engine.py:158-174) for a batch: one token of each
// of many requests (qfn_deltanet_step_batch), their states in slots of a pool,
// and the token-by-token recurrence over short sequences that
// qfn_deltanet_chunk uses below its crossover (dn_recurrence).
//
// Per row and value head, in fp32:
//   q = l2norm(q) / sqrt(dk), k = l2norm(k)   (l2norm: x * rsqrt(sum x^2 + 1e-6))
//   S = exp(g) S;  d = beta (v - S^T k);  S = S + k d^T;  out = bf16(S^T q)
//
// What bounds it: the state, 4 dk dv bytes read and written per row and head
// (2.1 MB each way for 32 heads of 128 x 128), against 7 flops per element.
// Every column of S is on its own, so CTA = (row, head, 32 columns): 128
// threads, a thread holds 4 neighbouring columns of dk / 16 rows in registers
// as float4 (a warp reads four 128-byte row pieces per instruction), all of
// them requested before anything else is.  The two sums over dk run over a
// thread's rows, then two shuffles and four warps through shared memory in a
// fixed order: results do not depend on the batch.
//
// Measured: 64 rows of 32 heads of 128 x 128 in 45 to 47 us, 5.8 to 6.0 TB/s; one
// row in 2.9 us in a graph.  The states go past the caches (__ldcs, __stcs): 50 us
// with plain loads and stores where these take 45.
#include "deltanet_batch.cuh"
#include "deltanet_chunk.cuh"

namespace qfn {

constexpr int kDbThreads = 128;
constexpr int kDbCols = 32;

// q (scaled) and k of one token and head into shared memory, normalised.
template <int DK>
__device__ __forceinline__ void dn_load_qk(const uint16_t* q, const uint16_t* k, float q_scale, float* qs, float* ks) {
  // warps 0 and 2 hold q, warps 1 and 3 k (2 and 3 repeat the sum and store nothing)
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint16_t* src = (w & 1) ? k : q;
  float x[DK / 32], acc = 0.f;
#pragma unroll
  for (int i = 0; i < DK / 32; ++i) {
    x[i] = bf16_bits_to_f32(src[i * 32 + lane]);
    acc = fmaf(x[i], x[i], acc);
  }
  acc = warp_sum(acc);
  const float r = rsqrtf(acc + 1e-6f);
  if (w < 2) {
    float* dst = w ? ks : qs;
#pragma unroll
    for (int i = 0; i < DK / 32; ++i) dst[i * 32 + lane] = w ? x[i] * r : (x[i] * r) / q_scale;
  }
}

__device__ __forceinline__ void dn_fold(float4& a) {   // sum over the warp's four row groups
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) {
    a.x += __shfl_xor_sync(0xffffffffu, a.x, o);
    a.y += __shfl_xor_sync(0xffffffffu, a.y, o);
    a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
    a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
  }
}

// One token: s[] is the thread's part of S; qs, ks hold q and k (visible to
// the block); writes 32 outputs.  Ends with the block past its last read of
// qs and ks.
template <int DK>
__device__ __forceinline__ void dn_token(float4 (&s)[DK / 16], const float* qs, const float* ks, float (*red)[2][kDbCols],
                                         float decay, float beta, const uint16_t* v, uint16_t* out) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, c4 = lane & 7, row0 = w * 4 + (lane >> 3);
  float4 kv = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int p = 0; p < DK / 16; ++p) {
    const float kk = ks[p * 16 + row0];
    s[p].x *= decay; s[p].y *= decay; s[p].z *= decay; s[p].w *= decay;
    kv.x = fmaf(s[p].x, kk, kv.x); kv.y = fmaf(s[p].y, kk, kv.y);
    kv.z = fmaf(s[p].z, kk, kv.z); kv.w = fmaf(s[p].w, kk, kv.w);
  }
  dn_fold(kv);
  if (lane < 8) *reinterpret_cast<float4*>(&red[w][0][c4 * 4]) = kv;
  __syncthreads();
  float4 d = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 a = *reinterpret_cast<const float4*>(&red[i][0][c4 * 4]);
    d.x += a.x; d.y += a.y; d.z += a.z; d.w += a.w;
  }
  d.x = (bf16_bits_to_f32(v[c4 * 4]) - d.x) * beta;
  d.y = (bf16_bits_to_f32(v[c4 * 4 + 1]) - d.y) * beta;
  d.z = (bf16_bits_to_f32(v[c4 * 4 + 2]) - d.z) * beta;
  d.w = (bf16_bits_to_f32(v[c4 * 4 + 3]) - d.w) * beta;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int p = 0; p < DK / 16; ++p) {
    const float kk = ks[p * 16 + row0], qq = qs[p * 16 + row0];
    s[p].x = fmaf(kk, d.x, s[p].x); s[p].y = fmaf(kk, d.y, s[p].y);
    s[p].z = fmaf(kk, d.z, s[p].z); s[p].w = fmaf(kk, d.w, s[p].w);
    o.x = fmaf(s[p].x, qq, o.x); o.y = fmaf(s[p].y, qq, o.y);
    o.z = fmaf(s[p].z, qq, o.z); o.w = fmaf(s[p].w, qq, o.w);
  }
  dn_fold(o);
  if (lane < 8) *reinterpret_cast<float4*>(&red[w][1][c4 * 4]) = o;
  __syncthreads();
  if (threadIdx.x < kDbCols) {
    const int c = threadIdx.x;
    out[c] = dn_bf16_bits(((red[0][1][c] + red[1][1][c]) + red[2][1][c]) + red[3][1][c]);
  }
}

template <int DK>
__device__ __forceinline__ void dn_store_state(const float4 (&s)[DK / 16], float* S, int dv) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, c4 = lane & 7, row0 = w * 4 + (lane >> 3);
#pragma unroll
  for (int p = 0; p < DK / 16; ++p)
    __stcs(reinterpret_cast<float4*>(S + static_cast<int64_t>(p * 16 + row0) * dv + c4 * 4), s[p]);
}

template <int DK>
__device__ __forceinline__ void dn_load_state(float4 (&s)[DK / 16], const float* S, int dv) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, c4 = lane & 7, row0 = w * 4 + (lane >> 3);
#pragma unroll
  for (int p = 0; p < DK / 16; ++p)
    s[p] = S ? __ldcs(reinterpret_cast<const float4*>(S + static_cast<int64_t>(p * 16 + row0) * dv + c4 * 4))
             : make_float4(0.f, 0.f, 0.f, 0.f);
}

// One token of each row.  index: the row's slot (null: the row itself);
// negative: a padding row (out = 0, no state).  A slot outside the pool, or
// one that an earlier row of the batch names, is not touched (out = NaN).
template <int DK>
__global__ void __launch_bounds__(kDbThreads) deltanet_step_batch_kernel(const DnRows a, const int32_t* index,
                                                                         int64_t n_slots) {
  __shared__ float qs[DK], ks[DK];
  __shared__ __align__(16) float red[4][2][kDbCols];
  const int cb = a.dv / kDbCols;
  const int c0 = static_cast<int>(blockIdx.x % cb) * kDbCols;
  const int h = static_cast<int>(blockIdx.x / cb % a.heads);
  const int64_t row = blockIdx.x / cb / a.heads;
  pdl_wait();   // the state may come from the kernel before
  const int64_t slot = index ? index[row] : row;
  uint16_t* out = a.out + (row * a.heads + h) * a.dv + c0;
  const bool inside = slot >= 0 && slot < n_slots;
  const int64_t at = ((slot * a.heads + h) * DK) * a.dv + c0;
  float4 s[DK / 16];
  if (inside) dn_load_state<DK>(s, a.s_in + at, a.dv);
  int again = 0;
  if (index && inside)
    for (int64_t i = threadIdx.x; i < row; i += kDbThreads) again |= index[i] == slot;
  if (inside)
    dn_load_qk<DK>(a.q + row * a.q_row + h / a.ratio * a.q_head, a.k + row * a.k_row + h / a.ratio * a.k_head,
                   a.q_scale, qs, ks);
  if (__syncthreads_or(again) || !inside) {
    if (threadIdx.x < kDbCols) out[threadIdx.x] = slot < 0 ? 0 : 0x7fc0;
    return;
  }
  dn_token<DK>(s, qs, ks, red, expf(a.g[row * a.g_row + h * a.g_head]),
               bf16_bits_to_f32(a.beta[row * a.b_row + h * a.b_head]), a.v + row * a.v_row + h * a.v_head + c0, out);
  dn_store_state<DK>(s, a.s_out + at, a.dv);
}

// The recurrence over the tokens of each sequence, one after the other.
template <int DK>
__global__ void __launch_bounds__(kDbThreads) deltanet_recurrence_kernel(const DnRows a, const int32_t* cu,
                                                                         int64_t n_seqs, int64_t tokens) {
  __shared__ float qs[2][DK], ks[2][DK];
  __shared__ __align__(16) float red[4][2][kDbCols];
  const int cb = a.dv / kDbCols;
  const int c0 = static_cast<int>(blockIdx.x % cb) * kDbCols;
  const int h = static_cast<int>(blockIdx.x / cb % a.heads);
  const int64_t seq = blockIdx.x / cb / a.heads;
  pdl_wait();
  const int64_t at = ((seq * a.heads + h) * DK) * a.dv + c0;
  float4 s[DK / 16];
  dn_load_state<DK>(s, a.s_in ? a.s_in + at : nullptr, a.dv);
  int64_t t0 = 0, t1 = 0;
  if (!cu) {
    t0 = seq * (tokens / n_seqs);
    t1 = t0 + tokens / n_seqs;
  } else if (dn_plan_ok(cu, n_seqs, tokens)) {
    t0 = cu[seq];
    t1 = cu[seq + 1];
  } else {   // sequence bounds that do not rise: no token is touched, the state says so
#pragma unroll
    for (int p = 0; p < DK / 16; ++p) s[p] = make_float4(CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F);
  }
  const uint16_t* q = a.q + h / a.ratio * a.q_head;
  const uint16_t* k = a.k + h / a.ratio * a.k_head;
  for (int64_t t = t0; t < t1; ++t) {
    const int b = static_cast<int>(t & 1);   // two buffers: a slow warp may still read the last token's
    dn_load_qk<DK>(q + t * a.q_row, k + t * a.k_row, a.q_scale, qs[b], ks[b]);
    __syncthreads();
    dn_token<DK>(s, qs[b], ks[b], red, expf(a.g[t * a.g_row + h * a.g_head]),
                 bf16_bits_to_f32(a.beta[t * a.b_row + h * a.b_head]), a.v + t * a.v_row + h * a.v_head + c0,
                 a.out + (t * a.heads + h) * a.dv + c0);
  }
  dn_store_state<DK>(s, a.s_out + at, a.dv);
}

int dn_rows_check(const char* what, const uint16_t* q, const uint16_t* k, const uint16_t* v, const float* g,
                  const uint16_t* beta, const int64_t* strides, const float* s_in, float* s_out, uint16_t* out,
                  int64_t rows, int64_t states, int n_heads, int n_key_heads, int dk, int dv, DnRows* r) {
  QFN_REQUIRE((rows == 0 || (q && k && v && g && beta && out)) && strides && (states == 0 || s_out),
              QFN_ERR_INVALID_ARG, "%s: null pointer", what);
  QFN_REQUIRE(n_heads >= 1 && n_key_heads >= 1 && n_heads % n_key_heads == 0, QFN_ERR_INVALID_ARG,
              "%s: n_heads=%d must be a multiple of n_key_heads=%d", what, n_heads, n_key_heads);
  QFN_REQUIRE((dk == 64 || dk == 128 || dk == 256) && dv >= 32 && dv <= 4096 && dv % 32 == 0, QFN_ERR_UNSUPPORTED,
              "%s: dk=%d (64, 128 or 256) and dv=%d (a multiple of 32, at most 4096) unsupported", what, dk, dv);
  QFN_REQUIRE(aligned(s_in, 16) && aligned(s_out, 16), QFN_ERR_ALIGNMENT, "%s: states must be 16-byte aligned", what);
  r->q = q; r->k = k; r->v = v; r->g = g; r->beta = beta;
  r->q_row = strides[0]; r->q_head = strides[1]; r->k_row = strides[2]; r->k_head = strides[3];
  r->v_row = strides[4]; r->v_head = strides[5]; r->g_row = strides[6]; r->g_head = strides[7];
  r->b_row = strides[8]; r->b_head = strides[9];
  r->out = out; r->s_in = s_in; r->s_out = s_out;
  r->heads = n_heads; r->ratio = n_heads / n_key_heads; r->dv = dv;
  r->q_scale = static_cast<float>(sqrt(static_cast<double>(dk)));
  return QFN_OK;
}

namespace {

bool clash(const void* x, uintptr_t x_bytes, const void* y, uintptr_t y_bytes) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
  return x && y && x_bytes && y_bytes && a < b + y_bytes && b < a + x_bytes;
}

// States that overlap without being the same would be read after they were written.
bool states_clash(const float* in, const float* out, int64_t n) {
  const uintptr_t bytes = static_cast<uintptr_t>(n) * sizeof(float);
  return in != out && clash(in, bytes, out, bytes);
}

// Outputs are written while other blocks still read states.
bool out_clash(const DnRows& a, int64_t rows, int64_t states, int dk) {
  const uintptr_t out = static_cast<uintptr_t>(rows) * a.heads * a.dv * sizeof(uint16_t),
                  S = static_cast<uintptr_t>(states) * a.heads * dk * a.dv * sizeof(float);
  return clash(a.out, out, a.s_in, S) || clash(a.out, out, a.s_out, S);
}

// The grid waits for the kernel before it (pdl_wait) and never releases the
// next one early: that one may read the state before its own wait.
template <typename Kernel, typename... Args>
int launch(const char* what, Kernel kernel, int64_t blocks, qfn_stream_t stream, Args... args) {
  QFN_REQUIRE(blocks <= 0x7fffffff, QFN_ERR_UNSUPPORTED, "%s: too many rows", what);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kDbThreads);
  cfg.stream = as_stream(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return set_error(QFN_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace

}  // namespace qfn

using namespace qfn;

extern "C" int qfn_deltanet_step_batch(const uint16_t* q, const uint16_t* k, const uint16_t* v, const float* g,
                                       const uint16_t* beta, const int64_t* strides, const int32_t* state_index,
                                       int64_t n_slots, const float* state_in, float* state_out, uint16_t* out,
                                       int64_t rows, int n_heads, int n_key_heads, int dk, int dv,
                                       qfn_stream_t stream) {
  constexpr const char* what = "qfn_deltanet_step_batch";
  DnRows a;
  int rc = dn_rows_check(what, q, k, v, g, beta, strides, state_in, state_out, out, rows, rows, n_heads,
                         n_key_heads, dk, dv, &a);
  if (rc) return rc;
  QFN_REQUIRE(rows == 0 || state_in, QFN_ERR_INVALID_ARG, "%s: null pointer", what);
  QFN_REQUIRE(rows >= 0 && n_slots >= 1 && (state_index || rows <= n_slots), QFN_ERR_INVALID_ARG,
              "%s: rows=%lld, n_slots=%lld (a slot for each row without state_index)", what,
              static_cast<long long>(rows), static_cast<long long>(n_slots));
  QFN_REQUIRE(!states_clash(state_in, state_out, n_slots * n_heads * dk * dv), QFN_ERR_INVALID_ARG,
              "%s: state_in and state_out overlap", what);
  QFN_REQUIRE(!out_clash(a, rows, n_slots, dk), QFN_ERR_INVALID_ARG, "%s: out overlaps a state", what);
  if (rows == 0) return QFN_OK;
  DeviceInfo* dev;
  rc = current_device(&dev);
  if (rc) return rc;
  const int64_t blocks = rows * n_heads * (dv / kDbCols);
  auto kernel = dk == 64 ? deltanet_step_batch_kernel<64>
                         : dk == 128 ? deltanet_step_batch_kernel<128> : deltanet_step_batch_kernel<256>;
  return launch(what, kernel, blocks, stream, a, state_index, n_slots);
}

extern "C" size_t qfn_deltanet_chunk_workspace(int64_t tokens, int64_t n_seqs, int n_heads, int n_key_heads, int dk,
                                               int dv) {
  if (tokens < 0 || n_seqs < 1 || n_heads < 1 || n_key_heads < 1 || dk < 1 || dv < 1 ||
      !dn_chunk_takes(tokens, n_seqs, n_heads, dk, dv))
    return 0;
  return dn_chunk_workspace(tokens, n_seqs, n_heads, n_key_heads, dk);
}

extern "C" int qfn_deltanet_chunk(const uint16_t* q, const uint16_t* k, const uint16_t* v, const float* g,
                                  const uint16_t* beta, const int64_t* strides, const int32_t* cu_seqlens,
                                  int64_t n_seqs, int64_t tokens, const float* state_in, float* state_out,
                                  uint16_t* out, int n_heads, int n_key_heads, int dk, int dv, void* workspace,
                                  size_t workspace_bytes, qfn_stream_t stream) {
  constexpr const char* what = "qfn_deltanet_chunk";
  DnRows a;
  int rc = dn_rows_check(what, q, k, v, g, beta, strides, state_in, state_out, out, tokens, n_seqs, n_heads,
                         n_key_heads, dk, dv, &a);
  if (rc) return rc;
  QFN_REQUIRE(n_seqs >= 0 && tokens >= 0 && (cu_seqlens || (n_seqs == 0 ? tokens == 0 : tokens % n_seqs == 0)),
              QFN_ERR_INVALID_ARG, "%s: tokens=%lld, n_seqs=%lld (equal lengths without cu_seqlens)", what,
              static_cast<long long>(tokens), static_cast<long long>(n_seqs));
  QFN_REQUIRE(!states_clash(state_in, state_out, n_seqs * n_heads * dk * dv), QFN_ERR_INVALID_ARG,
              "%s: state_in and state_out overlap", what);
  QFN_REQUIRE(tokens < (int64_t{1} << 31) - 64, QFN_ERR_UNSUPPORTED, "%s: tokens=%lld", what,
              static_cast<long long>(tokens));
  if (n_seqs == 0) return QFN_OK;
  const bool chunked = dn_chunk_takes(cu_seqlens ? tokens : tokens / n_seqs, n_seqs, n_heads, dk, dv);
  if (chunked) {
    const size_t need = dn_chunk_workspace(tokens, n_seqs, n_heads, n_key_heads, dk);
    QFN_REQUIRE(workspace && workspace_bytes >= need, QFN_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what,
                workspace ? workspace_bytes : size_t{0}, need);
    QFN_REQUIRE(aligned(workspace, 256), QFN_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", what);
    QFN_REQUIRE(aligned(out, 4), QFN_ERR_ALIGNMENT, "%s: out must be 4-byte aligned", what);
  }
  QFN_REQUIRE(!out_clash(a, tokens, n_seqs, dk), QFN_ERR_INVALID_ARG, "%s: out overlaps a state", what);
  DeviceInfo* dev;
  rc = current_device(&dev);
  if (rc) return rc;
  if (chunked) return dn_chunk(a, cu_seqlens, n_seqs, tokens, dk, *dev, workspace, stream);
  const int64_t blocks = n_seqs * n_heads * (dv / kDbCols);
  auto kernel = dk == 64 ? deltanet_recurrence_kernel<64>
                         : dk == 128 ? deltanet_recurrence_kernel<128> : deltanet_recurrence_kernel<256>;
  return launch(what, kernel, blocks, stream, a, cu_seqlens, n_seqs, tokens);
}
