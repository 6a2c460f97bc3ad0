// Attention of one new token a sequence over a batch's paged cache, the weights accumulated on request
// (sc_decode_attention). A block per (sequence, query head): its warps take the slots in turn, each with an online
// softmax of its own (running maximum m, sum l and output o, rescaled by 2^(m - m') when the maximum moves), joined in
// shared memory. With weights, a second kernel takes 2^(s - m) / l of every head at each slot.
#include <type_traits>

#include "pages.cuh"

namespace sc {
namespace da {

constexpr int WARPS = 8;

struct Args {
  Pages pages;
  const void* q;
  int64_t q_row, q_head;
  int q_heads, group, dim;
  float scale_log2;
  void* out;
  float* weight;
  int64_t weight_row;
  float2* stats;  // (batch, q_heads): maximum (log2 domain) and sum
  int* err;
};

// the score of one slot: a warp, lane l takes values l, l + 32, ...
template <typename T>
__device__ __forceinline__ float score(const float (&q)[8], const T* k, int dim, int lane) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < dim) s = fmaf(q[i], to_f32(k[lane + 32 * i]), s);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

template <typename T>
__global__ void __launch_bounds__(WARPS * 32) attend_kernel(const Args A) {
  __shared__ float s_m[WARPS], s_l[WARPS], s_o[WARPS][256];
  const int b = blockIdx.x, h = blockIdx.y, hk = h / A.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = length_of(A.pages, b, A.err);
  const T* q = static_cast<const T*>(A.q) + b * A.q_row + h * A.q_head;
  float qv[8], o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    qv[i] = lane + 32 * i < A.dim ? to_f32(q[lane + 32 * i]) * A.scale_log2 : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int mask = (1 << A.pages.shift) - 1;
  for (int s = warp; s < n; s += WARPS) {
    const int page = page_of(A.pages, b, s, A.err);
    if (page < 0) continue;
    const T* k = reinterpret_cast<const T*>(A.pages.k + page * A.pages.k_page + (s & mask) * A.pages.k_token + hk * A.pages.k_head);
    const T* v = reinterpret_cast<const T*>(A.pages.v + page * A.pages.v_page + (s & mask) * A.pages.v_token + hk * A.pages.v_head);
    const float x = score(qv, k, A.dim, lane), top = fmaxf(m, x);
    const float c = m == top ? 1.f : exp2f(m - top), p = exp2f(x - (top == -INFINITY ? 0.f : top));
    m = top;
    l = l * c + p;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < A.dim) o[i] = fmaf(p, to_f32(v[lane + 32 * i]), o[i] * c);
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int i = 0; i < 8; ++i) s_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w]);
  const float base = M == -INFINITY ? 0.f : M;
  for (int w = 0; w < WARPS; ++w) L += s_l[w] * exp2f(s_m[w] - base);
  for (int d = threadIdx.x; d < A.dim; d += WARPS * 32) {
    float r = 0.f;
    for (int w = 0; w < WARPS; ++w) r += s_o[w][d] * exp2f(s_m[w] - base);
    static_cast<T*>(A.out)[(int64_t(b) * A.q_heads + h) * A.dim + d] = from_f32<T>(L == 0.f ? 0.f : r / L);
  }
  if (threadIdx.x == 0) A.stats[int64_t(b) * A.q_heads + h] = make_float2(base, L);
}

// a warp a slot: every query head's probability there
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) weight_kernel(const Args A) {
  const int b = blockIdx.y, s = blockIdx.x * WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (s >= length_of(A.pages, b, nullptr)) return;
  const int page = page_of(A.pages, b, s, nullptr);
  if (page < 0) return;
  const int mask = (1 << A.pages.shift) - 1;
  float sum = 0.f;
  for (int h = 0; h < A.q_heads; ++h) {
    const T* q = static_cast<const T*>(A.q) + b * A.q_row + h * A.q_head;
    const T* k = reinterpret_cast<const T*>(A.pages.k + page * A.pages.k_page + (s & mask) * A.pages.k_token + h / A.group * A.pages.k_head);
    float qv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) qv[i] = lane + 32 * i < A.dim ? to_f32(q[lane + 32 * i]) * A.scale_log2 : 0.f;
    const float2 st = A.stats[int64_t(b) * A.q_heads + h];
    sum += exp2f(score(qv, k, A.dim, lane) - st.x) / st.y;
  }
  if (lane == 0) A.weight[b * A.weight_row + s] += sum;
}

}  // namespace da
}  // namespace sc

using namespace sc;

extern "C" size_t sc_decode_attention_workspace(const sc_kv_pages* kv, int q_heads) {
  if (check_pages(kv) || q_heads < 1 || q_heads % kv->kv_heads) return 0;
  return size_t(kv->batch > 0 ? kv->batch : 1) * q_heads * sizeof(float2);
}

extern "C" int sc_decode_attention(const sc_kv_pages* kv, const void* q, int64_t q_row, int64_t q_head, int q_heads,
                                   float scale, void* out, void* workspace, size_t workspace_bytes, int* err,
                                   void* stream) {
  if (int rc = check_pages(kv)) return rc;
  if (kv->batch && (!q || !out || !workspace)) return SC_ERR_ARG;
  if (q_heads < 1 || q_heads % kv->kv_heads || q_heads > 65535) return SC_ERR_SHAPE;
  if (((q_row | q_head) & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 15))
    return SC_ERR_ALIGN;
  if (workspace_bytes < sc_decode_attention_workspace(kv, q_heads)) return SC_ERR_WORKSPACE;
  if (kv->batch == 0) return SC_OK;
  da::Args A{};
  A.pages = pages_of(*kv);
  A.q = q, A.q_row = q_row, A.q_head = q_head;
  A.q_heads = q_heads, A.group = q_heads / kv->kv_heads, A.dim = kv->head_dim;
  A.scale_log2 = scale * 1.4426950408889634f;
  A.out = out, A.weight = kv->weight, A.weight_row = kv->weight_row;
  A.stats = static_cast<float2*>(workspace);
  A.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto run = [&](auto t) {
    using T = decltype(t);
    da::attend_kernel<T><<<dim3(kv->batch, q_heads), da::WARPS * 32, 0, s>>>(A);
    if (A.weight)
      da::weight_kernel<T><<<dim3(unsigned(ceil_div(int64_t(kv->max_pages) * kv->page, da::WARPS)), kv->batch), da::WARPS * 32, 0, s>>>(A);
  };
  if (kv->dtype == SC_BF16) run(__nv_bfloat16{});
  else run(__half{});
  if (cudaError_t e = cudaGetLastError()) return cuda_failed(e, "decode attention launch");
  return SC_OK;
}
