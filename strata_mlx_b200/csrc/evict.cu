// Eviction from a paged cache by accumulated attention weight (sc_evict).
//
//   plan_kernel  a block a sequence: each slot's key is its class (kept by its place or not) and its weight as an
//                unsigned integer of the same order; four passes over eight bits each, a histogram a pass, find the
//                key of the last slot that stays. Then one pass in slot order lists the holes (evicted slots below
//                the budget) and the movers (kept slots past it): as many of one as of the other.
//   move_kernel  mover i's keys, values, weight and position into hole i. Sources lie at or past the budget and
//                destinations below it, so no row is read that another block writes, and the order is free.
#include "pages.cuh"

namespace sc {
namespace ev {

constexpr int THREADS = 1024;
constexpr int MOVE_WARPS = 8;

struct Args {
  Pages pages;
  const float* weight;
  const int32_t *position, *seen;
  int64_t weight_row, position_row;
  int keep, sinks, recent, cap, row16;  // cap: entries of a sequence's lists; row16: 16-byte words of a head
  int kv_heads;
  float* weight_out;
  int32_t *position_out, *lengths_out;
  int64_t weight_out_row, position_out_row;
  int32_t *count, *src, *dst;  // (batch), (batch, cap), (batch, cap)
  int* err;
};

// weights as integers of the same order: the largest float has the largest integer, a NaN above all
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 and 0 are equal
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int block_sum(int v, int* sh) {  // over the block, the same value in every thread
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = sh[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  __syncthreads();
  return t;
}

// threads before this one with v set, and the block's count
__device__ __forceinline__ int block_rank(bool v, int* sh, int& total) {
  const unsigned m = __ballot_sync(0xffffffffu, v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) sh[warp] = __popc(m);
  __syncthreads();
  const int mine = sh[lane];
  int x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  const int before = __shfl_sync(0xffffffffu, x - mine, warp);
  total = __shfl_sync(0xffffffffu, x, 31);
  __syncthreads();
  return before + __popc(m & ((1u << lane) - 1));
}

__global__ void __launch_bounds__(THREADS) plan_kernel(const Args A) {
  __shared__ int sh[32], hist[256], pick[2];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int n = length_of(A.pages, b, A.err);
  const float* w = A.weight + b * A.weight_row;
  const int32_t* pos = A.position + b * A.position_row;
  float* wo = A.weight_out + b * A.weight_out_row;
  int32_t* po = A.position_out + b * A.position_out_row;
  __syncthreads();  // lengths_out may be the lengths themselves
  if (tid == 0) A.lengths_out[b] = min(n, A.keep);
  if (n <= A.keep) {
    if (tid == 0) A.count[b] = 0;
    for (int s = tid; s < n; s += THREADS) {
      const float x = w[s];
      const int32_t p = pos[s];
      wo[s] = x;
      po[s] = p;
    }
    return;
  }
  const int64_t from = int64_t(A.seen[b]) - A.recent;
  auto safe = [&](int s) { return pos[s] < A.sinks || pos[s] >= from; };
  int c = 0;
  for (int s = tid; s < n; s += THREADS) c += safe(s);
  const int safes = block_sum(c, sh);
  // the class in which the last slot that stays is found, and how many of it stay
  const bool cls = safes >= A.keep;
  int want = cls ? A.keep : A.keep - safes;
  uint32_t key = 0, known = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
    __syncthreads();
    for (int s = tid; s < n; s += THREADS)
      if (safe(s) == cls) {
        const uint32_t k = order_of(w[s]);
        if ((k & known) == key) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
    __syncthreads();
    if (tid == 0) {
      int above = 0, d = 255;
      while (d > 0 && above + hist[d] < want) above += hist[d--];
      pick[0] = d, pick[1] = above;
    }
    __syncthreads();
    key |= uint32_t(pick[0]) << shift;
    known |= 255u << shift;
    want -= pick[1];
    __syncthreads();
  }
  // `want` of the slots with this key stay: the lowest ones
  int ties = 0, holes = 0, movers = 0;
  for (int s0 = 0; s0 < n; s0 += THREADS) {
    const int s = s0 + tid;
    bool stays = false, tie = false;
    if (s < n) {
      const bool sf = safe(s);
      const uint32_t k = order_of(w[s]);
      tie = sf == cls && k == key;
      stays = sf == cls ? k > key : sf;
    }
    int total;
    const int at = block_rank(tie, sh, total);
    if (tie) stays = ties + at < want;
    ties += total;
    const bool hole = s < A.keep && s < n && !stays, mover = s >= A.keep && stays;
    const int hr = block_rank(hole, sh, total);
    if (hole) A.dst[int64_t(b) * A.cap + holes + hr] = s;
    holes += total;
    const int mr = block_rank(mover, sh, total);
    if (mover) A.src[int64_t(b) * A.cap + movers + mr] = s;
    movers += total;
    if (s < A.keep && stays) {
      const float x = w[s];
      const int32_t p = pos[s];
      wo[s] = x;
      po[s] = p;
    }
  }
  if (tid == 0) A.count[b] = movers;
}

// a warp a row
__global__ void __launch_bounds__(MOVE_WARPS * 32) move_kernel(const Args A) {
  const int b = blockIdx.y, lane = threadIdx.x & 31, count = A.count[b];
  const int mask = (1 << A.pages.shift) - 1;
  for (int i = blockIdx.x * MOVE_WARPS + (threadIdx.x >> 5); i < count; i += gridDim.x * MOVE_WARPS) {
    const int s = A.src[int64_t(b) * A.cap + i], d = A.dst[int64_t(b) * A.cap + i];
    const int ps = page_of(A.pages, b, s, A.err), pd = page_of(A.pages, b, d, A.err);
    if (lane == 0) {
      A.weight_out[b * A.weight_out_row + d] = A.weight[b * A.weight_row + s];
      A.position_out[b * A.position_out_row + d] = A.position[b * A.position_row + s];
    }
    if (ps < 0 || pd < 0) continue;
    const Pages& p = A.pages;
    const char* ks = p.k + ps * p.k_page + (s & mask) * p.k_token;
    const char* vs = p.v + ps * p.v_page + (s & mask) * p.v_token;
    char* kd = const_cast<char*>(p.k) + pd * p.k_page + (d & mask) * p.k_token;
    char* vd = const_cast<char*>(p.v) + pd * p.v_page + (d & mask) * p.v_token;
    for (int j = lane; j < A.kv_heads * A.row16; j += 32) {
      const int h = j / A.row16, e = 16 * (j % A.row16);
      *reinterpret_cast<uint4*>(kd + h * p.k_head + e) = *reinterpret_cast<const uint4*>(ks + h * p.k_head + e);
      *reinterpret_cast<uint4*>(vd + h * p.v_head + e) = *reinterpret_cast<const uint4*>(vs + h * p.v_head + e);
    }
  }
}

// entries of a sequence's lists: holes lie below `keep`, movers at or past it
inline int64_t list_cap(const sc_kv_pages& c, int keep) {
  const int64_t slots = int64_t(c.max_pages) * c.page;
  return slots > keep ? (keep < slots - keep ? keep : slots - keep) : 0;
}

}  // namespace ev
}  // namespace sc

using namespace sc;

extern "C" size_t sc_evict_workspace(const sc_kv_pages* kv, int keep) {
  if (check_pages(kv) || keep < 0) return 0;
  const size_t n = kv->batch > 0 ? kv->batch : 1;
  return 4 * (n + 2 * n * size_t(ev::list_cap(*kv, keep))) + 16;
}

extern "C" int sc_evict(const sc_kv_pages* kv, const int32_t* seen, int keep, int sinks, int recent, float* weight_out,
                        int64_t weight_out_row, int32_t* position_out, int64_t position_out_row, int32_t* lengths_out,
                        void* workspace, size_t workspace_bytes, int* err, void* stream) {
  if (int rc = check_pages(kv)) return rc;
  if (keep < 0 || sinks < 0 || recent < 0 ||
      (kv->batch && (!kv->weight || !kv->position || !seen || !weight_out || !position_out || !lengths_out || !workspace)))
    return SC_ERR_ARG;
  if (int64_t(sinks) + recent > keep) return SC_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return SC_ERR_ALIGN;
  if (workspace_bytes < sc_evict_workspace(kv, keep)) return SC_ERR_WORKSPACE;
  if (kv->batch == 0) return SC_OK;
  ev::Args A{};
  A.pages = pages_of(*kv);
  A.weight = kv->weight, A.weight_row = kv->weight_row;
  A.position = kv->position, A.position_row = kv->position_row;
  A.seen = seen, A.keep = keep, A.sinks = sinks, A.recent = recent;
  A.cap = int(ev::list_cap(*kv, keep));
  A.row16 = kv->head_dim / 8, A.kv_heads = kv->kv_heads;
  A.weight_out = weight_out, A.weight_out_row = weight_out_row;
  A.position_out = position_out, A.position_out_row = position_out_row;
  A.lengths_out = lengths_out;
  A.count = static_cast<int32_t*>(workspace);
  A.src = A.count + kv->batch;
  A.dst = A.src + int64_t(kv->batch) * A.cap;
  A.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ev::plan_kernel<<<kv->batch, ev::THREADS, 0, s>>>(A);
  if (A.cap) {
    const int64_t blocks = ceil_div(A.cap, ev::MOVE_WARPS);
    ev::move_kernel<<<dim3(unsigned(blocks < 1024 ? blocks : 1024), kv->batch), ev::MOVE_WARPS * 32, 0, s>>>(A);
  }
  if (cudaError_t e = cudaGetLastError()) return cuda_failed(e, "evict launch");
  return SC_OK;
}
