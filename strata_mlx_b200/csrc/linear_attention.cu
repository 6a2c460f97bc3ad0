// Linear attention with a decay a head and token as its recurrence,
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t:
// over prompts that the tensor cores do not take (linear_chunk.cu takes the others), and one token a sequence.
#include "linear.cuh"

namespace sc {
namespace la {

constexpr int FEW = 8;  // tokens that the recurrence takes
constexpr int COLS = 32, PARTS = 8, MAXK = 128, PER = MAXK / PARTS, GROUP = 16;

// A block per (sequence, value head, 32 value dimensions) holds its columns of S in registers, a thread 1/8 of a column,
// and walks the tokens, GROUP of them at a time through shared memory; the eight parts of the group's outputs meet
// there. Bound by the chain of tokens: 0.31 us each at 128 x 128.
template <typename T>
__global__ void __launch_bounds__(COLS * PARTS) recurrent_kernel(const sc_linear A) {
  __shared__ __align__(16) float s_q[GROUP][MAXK], s_k[GROUP][MAXK];  // part p's rows p, p + 8, ... together
  __shared__ float s_v[GROUP][COLS], s_o[GROUP][PARTS][COLS], s_a[GROUP];
  __shared__ bool s_near[GROUP];
  const int h = blockIdx.x, b = blockIdx.y, hk = h / (A.v_heads / A.k_heads), tid = threadIdx.x;
  const int c = tid % COLS, col = blockIdx.z * COLS + c, part = tid / COLS;
  const bool live = col < A.v_dim;
  int n = A.tokens;
  if (A.lengths) n = min(max(A.lengths[b], 0), n);
  const int64_t at = (int64_t(b) * A.v_heads + h) * A.k_dim * A.v_dim + col;
  float S[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = part + PARTS * i;
    S[i] = live && r < A.k_dim && A.state_in ? A.state_in[at + int64_t(r) * A.v_dim] : 0.f;
  }
  const T* q = static_cast<const T*>(A.q) + b * A.q_row + hk * A.q_head;
  const T* k = static_cast<const T*>(A.k) + b * A.k_row + hk * A.k_head;
  const T* v = static_cast<const T*>(A.v) + b * A.v_row + h * A.v_head;
  const float* decay = A.decay + b * A.decay_row + h * A.decay_head;
  T* out = static_cast<T*>(A.out) + (int64_t(b) * A.tokens * A.v_heads + h) * A.v_dim;
  const int64_t row = int64_t(A.v_heads) * A.v_dim;
  for (int t0 = 0; t0 < n; t0 += GROUP) {
    const int m = min(GROUP, n - t0);
    for (int e = tid; e < m * MAXK; e += COLS * PARTS) {
      const int t = e / MAXK, d = e % MAXK, to = d % PARTS * PER + d / PARTS;
      const bool in = d < A.k_dim;
      s_q[t][to] = in ? to_f32(q[(t0 + t) * A.q_token + d]) * A.scale : 0.f;
      s_k[t][to] = in ? to_f32(k[(t0 + t) * A.k_token + d]) : 0.f;
    }
    for (int t = part; t < m; t += PARTS) s_v[t][c] = live ? to_f32(v[(t0 + t) * A.v_token + col]) : 0.f;
    if (tid < m) {
      // S + (exp(g) - 1) S: near 1 the decay itself would carry a rounding that every later token repeats. A decay
      // below 1/2 multiplies S alone, or the difference would cancel.
      const float g = decay[(t0 + tid) * A.decay_token];
      s_near[tid] = g > -0.69314718f;
      s_a[tid] = s_near[tid] ? expm1f(g) : expf(g);
    }
    __syncthreads();
    for (int t = 0; t < m; ++t) {
      const float a = s_a[t], x = s_v[t][c];
      const bool near = s_near[t];
      float o = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        S[i] = fmaf(s_k[t][part * PER + i], x, near ? fmaf(a, S[i], S[i]) : a * S[i]);
        o = fmaf(s_q[t][part * PER + i], S[i], o);
      }
      s_o[t][part][c] = o;
    }
    __syncthreads();
    for (int t = part; t < m; t += PARTS) {
      float r = 0.f;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) r += s_o[t][i][c];
      if (live) out[(t0 + t) * row + col] = from_f32<T>(r);
    }
  }
  if (live)
    for (int t = n + part; t < A.tokens; t += PARTS) out[t * row + col] = from_f32<T>(0.f);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = part + PARTS * i;
    if (live && r < A.k_dim) A.state_out[at + int64_t(r) * A.v_dim] = S[i];
  }
}

// One token a sequence. The states' bytes bound it, read and written once: a block per (sequence, value head, 32 value
// dimensions), a thread four of them in every 32nd row, all its rows' loads in flight before the first is used. The
// rows' parts of the output meet by shuffles and in shared memory. Blocks of 32 columns (128-byte pieces of rows)
// give one sequence's 16 heads four blocks each. Measured: 64 sequences of 32 heads, 128 x 128, 47 to 52 us (5.2 to 5.7
// TB/s of the 6.45 that a copy reaches); one sequence of 16 heads 2.6 us.
constexpr int STEP_THREADS = 256, STEP_ROWS = STEP_THREADS / 8;

template <typename T>
__global__ void __launch_bounds__(STEP_THREADS) step_kernel(const sc_linear A) {
  __shared__ float4 s_o[STEP_THREADS / 32][8];
  const int h = blockIdx.y, b = blockIdx.z, hk = h / (A.v_heads / A.k_heads);
  const int col = blockIdx.x * 32 + 4 * (threadIdx.x & 7), row = threadIdx.x >> 3;
  const bool live = col < A.v_dim;
  const int64_t at = (int64_t(b) * A.v_heads + h) * A.k_dim * A.v_dim + col;
  const T* q = static_cast<const T*>(A.q) + b * A.q_row + hk * A.q_head;
  const T* k = static_cast<const T*>(A.k) + b * A.k_row + hk * A.k_head;
  float4 S[MAXK / STEP_ROWS];
  float kr[MAXK / STEP_ROWS], qr[MAXK / STEP_ROWS];
#pragma unroll
  for (int i = 0; i < MAXK / STEP_ROWS; ++i) {
    const int r = row + STEP_ROWS * i;
    kr[i] = r < A.k_dim ? to_f32(k[r]) : 0.f, qr[i] = r < A.k_dim ? to_f32(q[r]) : 0.f;
    S[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live && r < A.k_dim) S[i] = *reinterpret_cast<const float4*>(A.state_in + at + int64_t(r) * A.v_dim);
  }
  const float g = A.decay[b * A.decay_row + h * A.decay_head];
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const T*>(A.v) + b * A.v_row + h * A.v_head + col);
    const T* xv = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_f32(xv[e]);
  }
  // as in the recurrence over a prompt: the difference form near 1
  const bool near = g > -0.69314718f;
  const float a = near ? expm1f(g) : expf(g);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < MAXK / STEP_ROWS; ++i) {
    const int r = row + STEP_ROWS * i;
    float* s = reinterpret_cast<float*>(&S[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = fmaf(kr[i], v[e], near ? fmaf(a, s[e], s[e]) : a * s[e]);
    o.x = fmaf(qr[i], s[0], o.x), o.y = fmaf(qr[i], s[1], o.y), o.z = fmaf(qr[i], s[2], o.z), o.w = fmaf(qr[i], s[3], o.w);
    if (live && r < A.k_dim) *reinterpret_cast<float4*>(A.state_out + at + int64_t(r) * A.v_dim) = S[i];
  }
#pragma unroll
  for (int w = 8; w < 32; w <<= 1) {
    o.x += __shfl_xor_sync(0xffffffffu, o.x, w);
    o.y += __shfl_xor_sync(0xffffffffu, o.y, w);
    o.z += __shfl_xor_sync(0xffffffffu, o.z, w);
    o.w += __shfl_xor_sync(0xffffffffu, o.w, w);
  }
  if ((threadIdx.x & 31) < 8) s_o[threadIdx.x >> 5][threadIdx.x & 7] = o;
  __syncthreads();
  if (threadIdx.x < 8 && live) {
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < STEP_THREADS / 32; ++w) {
      const float4 p = s_o[w][threadIdx.x];
      o.x += p.x, o.y += p.y, o.z += p.z, o.w += p.w;
    }
    uint2 x;
    T* to = reinterpret_cast<T*>(&x);
    to[0] = from_f32<T>(o.x * A.scale), to[1] = from_f32<T>(o.y * A.scale);
    to[2] = from_f32<T>(o.z * A.scale), to[3] = from_f32<T>(o.w * A.scale);
    *reinterpret_cast<uint2*>(static_cast<T*>(A.out) + (int64_t(b) * A.v_heads + h) * A.v_dim + col) = x;
  }
}

inline int check(const sc_linear* a) {
  if (!a || a->batch < 0 || a->tokens < 0 || (a->batch && !a->state_out) ||
      (a->batch && a->tokens && (!a->q || !a->k || !a->v || !a->decay || !a->out)))
    return SC_ERR_ARG;
  if (a->dtype != SC_F16 && a->dtype != SC_BF16) return SC_ERR_DTYPE;
  if (a->k_heads < 1 || a->v_heads < 1 || a->v_heads % a->k_heads || a->k_dim < 8 || a->k_dim % 8 || a->k_dim > MAXK ||
      a->v_dim < 8 || a->v_dim % 8 || a->v_dim > 128 || a->batch > 65535 || a->v_heads > 65535)
    return SC_ERR_SHAPE;
  const int64_t strides = used(a->batch, a->q_row | a->k_row | a->v_row) |
                          used(a->tokens, a->q_token | a->k_token | a->v_token) |
                          used(a->k_heads, a->q_head | a->k_head) | used(a->v_heads, a->v_head);
  const uintptr_t p = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                      reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->out) |
                      reinterpret_cast<uintptr_t>(a->state_in) | reinterpret_cast<uintptr_t>(a->state_out);
  if ((strides & 7) || (p & 15)) return SC_ERR_ALIGN;
  return SC_OK;
}

int launch(const sc_linear& a, void* stream) {
  if (a.batch == 0) return SC_OK;
  const dim3 grid(unsigned(a.v_heads), unsigned(a.batch), unsigned((a.v_dim + COLS - 1) / COLS));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == SC_BF16) recurrent_kernel<__nv_bfloat16><<<grid, COLS * PARTS, 0, s>>>(a);
  else recurrent_kernel<__half><<<grid, COLS * PARTS, 0, s>>>(a);
  if (cudaError_t e = cudaGetLastError()) return cuda_failed(e, "linear attention launch");
  return SC_OK;
}

}  // namespace la
}  // namespace sc

using namespace sc;

// Prompts of bfloat16 go to the tensor cores. To the recurrence go a few tokens, which a chunk's products would mostly pad
// (16 heads of 128 x 128, one sequence of 8 tokens: 5.4 us, in a chunk 7.7; 32 heads, 16 sequences: 29.0 and 29.8 at 8
// tokens, 35.5 and 29.9 at 12), and what the chunks are not built for: broadcast axes (a map takes no stride of zero) and
// float16 (the states need bfloat16's exponents; queries, keys and values would enter as two bfloat16 terms each). That
// is slow for long ones: 0.31 us a token.
static bool chunked(const sc_linear& a) { return a.tokens > la::FEW && lc::takes(a); }

extern "C" size_t sc_linear_attention_workspace(const sc_linear* a) {
  if (la::check(a) || a->batch == 0) return 0;
  return chunked(*a) ? lc::workspace(*a) : 0;
}

extern "C" int sc_linear_attention(const sc_linear* a, void* workspace, size_t workspace_bytes, int* err, void* stream) {
  if (int rc = la::check(a)) return rc;
  if (a->batch == 0) return SC_OK;
  const size_t need = sc_linear_attention_workspace(a);
  if (need && !workspace) return SC_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return SC_ERR_ALIGN;
  if (workspace_bytes < need) return SC_ERR_WORKSPACE;
  if (chunked(*a)) return lc::launch(*a, workspace, err, static_cast<cudaStream_t>(stream));
  return la::launch(*a, stream);
}

extern "C" int sc_linear_attention_step(const sc_linear* a, void* stream) {
  if (int rc = la::check(a)) return rc;
  if (a->tokens != 1 || a->lengths) return SC_ERR_SHAPE;
  if (a->batch == 0) return SC_OK;
  if (!a->state_in) return SC_ERR_ARG;
  const dim3 grid(unsigned((a->v_dim + 31) / 32), unsigned(a->v_heads), unsigned(a->batch));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == SC_BF16) la::step_kernel<__nv_bfloat16><<<grid, la::STEP_THREADS, 0, s>>>(*a);
  else la::step_kernel<__half><<<grid, la::STEP_THREADS, 0, s>>>(*a);
  if (cudaError_t e = cudaGetLastError()) return cuda_failed(e, "linear attention step launch");
  return SC_OK;
}
