// Eviction from a paged cache by accumulated attention weight (sc_evict).
//
//   plan_kernel  a cluster of blocks a sequence, each with a stretch of its slots. A slot's key is its weight as an
//                unsigned integer of the same order, the largest integer where its place keeps it; keys stay in shared
//                memory. The key of the last slot that stays is found digit by digit below the bits that all keys
//                share: a histogram of 2048 digits a round in every block, summed over the cluster through distributed
//                shared memory. Then each warp ranks its slots in slot order (ballots, sums over warps and blocks) and
//                lists the holes (evicted slots below the budget) and the movers (kept slots past it): as many of one
//                as of the other. Latency bounds it: a round is two barriers and a walk over the histogram.
//   move_kernel  mover i's keys, values, weight and position into hole i. Sources lie at or past the budget and
//                destinations below it, so no row is read that another warp writes, and the order is free. Bandwidth
//                bounds it: a warp fetches the list entries and page ids of its rows at once and keeps four 16-byte
//                words a lane in flight.
#include <cooperative_groups.h>

#include <algorithm>

#include "pages.cuh"

namespace sc {
namespace ev {

namespace cg = cooperative_groups;

constexpr int THREADS = 1024, WARPS = THREADS / 32;
constexpr int BINS = 2048, BITS = 11;
constexpr int MAX_CLUSTER = 8;
constexpr int PER_BLOCK = 16384;  // slots of a block before the cluster grows
constexpr int MOST = 50 * 1024;   // slots a block can hold the keys of (200 KB); past 8 such blocks keys are made anew
constexpr int FETCH = 8;          // weights and positions a thread loads at a time
constexpr int MOVE_WARPS = 8;
constexpr uint32_t KEPT = 0xffffffffu;

struct Args {
  Pages pages;
  const float* weight;
  const int32_t *position, *seen;
  int64_t weight_row, position_row;
  int keep, sinks, recent, cap;  // cap: entries of a sequence's lists
  int heads, row16;              // a slot's keys: `heads` pieces of row16 16-byte words
  int hold;                      // slots whose keys a block holds
  float* weight_out;
  int32_t *position_out, *lengths_out;
  int64_t weight_out_row, position_out_row;
  int32_t *count, *src, *dst;  // (batch), (batch, cap), (batch, cap)
  int* err;
};

// weights as integers of the same order, a NaN above all others; 0 and KEPT are no weight's
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return KEPT - 1;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 and 0 are equal
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// sums and scans over a block; `sh` holds WARPS values
__device__ __forceinline__ int block_sum(int v, int* sh) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  const int t = __reduce_add_sync(0xffffffffu, sh[threadIdx.x & 31]);
  __syncthreads();
  return t;
}
__device__ __forceinline__ int warp_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

template <bool HELD>
__global__ void __launch_bounds__(THREADS) plan_kernel(const Args A) {
  extern __shared__ uint32_t s_key[];
  __shared__ int s_hist[2][BINS];
  __shared__ int s_warp[WARPS], s_pick[2];
  __shared__ int s_out[4][2];         // read by the other blocks, a pair for each use
  __shared__ uint32_t s_span[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int b = blockIdx.x / blocks, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  const int n = length_of(A.pages, b, A.err), keep = A.keep;
  const float* w = A.weight + b * A.weight_row;
  const int32_t* pos = A.position + b * A.position_row;
  float* wo = A.weight_out + b * A.weight_out_row;
  int32_t* po = A.position_out + b * A.position_out_row;
  // this block's slots, a whole number of them to each warp
  const int per = ((n + blocks - 1) / blocks + THREADS - 1) / THREADS * THREADS;
  const int s0 = min(n, rank * per), mine = min(n, s0 + per) - s0, span = per / WARPS;
  // a batch of this block's weights and positions, loaded together; those below the budget are copied at once (the
  // evicted among them are overwritten when their slots are filled)
  auto fetch = [&](auto f) {
    for (int i0 = tid; i0 < mine; i0 += FETCH * THREADS) {
      float x[FETCH];
      int32_t p[FETCH];
#pragma unroll
      for (int u = 0; u < FETCH; ++u)
        if (i0 + u * THREADS < mine) x[u] = w[s0 + i0 + u * THREADS], p[u] = pos[s0 + i0 + u * THREADS];
#pragma unroll
      for (int u = 0; u < FETCH; ++u) {
        const int i = i0 + u * THREADS;
        if (i < mine) {
          if (s0 + i < keep) wo[s0 + i] = x[u], po[s0 + i] = p[u];
          f(i, x[u], p[u]);
        }
      }
    }
  };
  if (n <= keep) {
    fetch([](int, float, int32_t) {});
    cluster.sync();  // lengths_out may be the lengths themselves
    if (rank == 0 && tid == 0) A.count[b] = 0, A.lengths_out[b] = n;
    return;
  }
  const int64_t from = int64_t(A.seen[b]) - A.recent;
  auto is_safe = [&](int32_t p) { return p < A.sinks || p >= from; };
  // every block's sum of a value, and the sums of the blocks before this one
  auto cluster_sum = [&](int v, int use, int& before) {
    const int t = block_sum(v, s_warp);
    before = 0;
    if (blocks == 1) return t;
    if (tid == 0) s_out[use][0] = t;
    cluster.sync();
    int all = 0;
    for (int r = 0; r < blocks; ++r) {
      const int x = *cluster.map_shared_rank(&s_out[use][0], r);
      if (r < rank) before += x;
      all += x;
    }
    return all;
  };
  // ---- keys: first with the kept places above all weights
  int c = 0;
  fetch([&](int i, float x, int32_t p) {
    const bool safe = is_safe(p);
    c += safe;
    if constexpr (HELD) s_key[i] = safe ? KEPT : order_of(x);
  });
  int none;
  const int safes = cluster_sum(c, 0, none);
  // more kept places than slots stay (positions that repeat): only they are ranked, by weight
  const bool crowded = safes > keep;
  auto make = [&](int i) -> uint32_t {
    const bool safe = is_safe(pos[s0 + i]);
    return crowded ? (safe ? order_of(w[s0 + i]) : 0u) : safe ? KEPT : order_of(w[s0 + i]);
  };
  if (HELD && crowded)
    for (int i = tid; i < mine; i += THREADS) s_key[i] = make(i);
  __syncthreads();
  auto key_at = [&](int i) { return HELD ? s_key[i] : make(i); };
  // ---- the bits that the keys below KEPT share
  uint32_t lo = KEPT, hi = 0;
  for (int i = tid; i < mine; i += THREADS) {
    const uint32_t k = key_at(i);
    if (k != KEPT) lo = min(lo, k), hi = max(hi, k);
  }
  lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
  if (tid == 0) s_span[0] = KEPT, s_span[1] = 0;
  __syncthreads();
  if (lane == 0) atomicMin(&s_span[0], lo), atomicMax(&s_span[1], hi);
  for (int i = tid; i < 2 * BINS; i += THREADS) s_hist[0][i] = 0;
  if (blocks > 1) cluster.sync();
  else __syncthreads();
  lo = KEPT, hi = 0;
  for (int r = 0; r < blocks; ++r) {
    lo = min(lo, *cluster.map_shared_rank(&s_span[0], r));
    hi = max(hi, *cluster.map_shared_rank(&s_span[1], r));
  }
  int want = crowded ? keep : keep - safes;  // how many of the slots below KEPT stay
  uint32_t key = KEPT;                       // slots above it stay, `want` of those at it
  if (want > 0) {
    int bits = hi > lo ? 32 - __clz(hi ^ lo) : 0;  // not shared
    key = bits < 32 ? (hi >> bits) << bits : 0u;
    for (int round = 0; bits > 0; ++round) {
      const int take = min(bits, BITS), shift = bits - take;
      const uint32_t known = bits < 32 ? ~0u << bits : 0u, digit = (1u << take) - 1;
      int* hist = s_hist[round & 1];
      for (int i = tid; i < mine; i += THREADS) {
        const uint32_t k = key_at(i);
        if (k != KEPT && (k & known) == key) atomicAdd(&hist[(k >> shift) & digit], 1);
      }
      if (blocks > 1) cluster.sync();
      else __syncthreads();
      // thread t takes the digits 2047 - 2t and 2046 - 2t, so that a scan counts from the top
      const int d1 = BINS - 1 - 2 * tid, d0 = d1 - 1;
      int n1 = 0, n0 = 0;
      for (int r = 0; r < blocks; ++r) {
        const int2 v = *reinterpret_cast<const int2*>(cluster.map_shared_rank(hist, r) + d0);
        n0 += v.x, n1 += v.y;
      }
      const int inc = warp_scan(n0 + n1);
      if (lane == 31) s_warp[warp] = inc;
      __syncthreads();
      const int sums = s_warp[lane], upto = __shfl_sync(0xffffffffu, warp_scan(sums) - sums, warp) + inc - n0 - n1;
      if (upto < want && want <= upto + n1) s_pick[0] = d1, s_pick[1] = upto;
      if (upto + n1 < want && want <= upto + n1 + n0) s_pick[0] = d0, s_pick[1] = upto + n1;
      // the other histogram, which no block reads any more, is the next round's
      for (int i = tid; i < BINS; i += THREADS) s_hist[(round + 1) & 1][i] = 0;
      __syncthreads();
      key |= uint32_t(s_pick[0]) << shift;
      want -= s_pick[1];
      bits = shift;
    }
  }
  // ---- in slot order: which of the slots at `key` stay, then the lists. Warp w has slots w span .. of this block's.
  const int w0 = warp * span, w1 = min(mine, w0 + span);
  auto each = [&](auto f) {
    for (int i = w0; i < w1; i += 32) f(i + lane, i + lane < w1);
  };
  int ties = 0;
  each([&](int i, bool in) { ties += __popc(__ballot_sync(0xffffffffu, in && key_at(i) == key)); });
  int before_blocks, at;
  const int all_ties = cluster_sum(lane == 0 ? ties : 0, 1, before_blocks);
  auto warps_before = [&](int v) {  // the sum over the warps before this one
    if (lane == 0) s_warp[warp] = v;
    __syncthreads();
    const int x = s_warp[lane];
    const int r = __shfl_sync(0xffffffffu, warp_scan(x) - x, warp);
    __syncthreads();
    return r;
  };
  const int stay_ties = key == KEPT ? all_ties : want;  // of KEPT all, or none are there
  const int tie0 = before_blocks + warps_before(ties);
  at = tie0;
  auto stays_at = [&](int i, bool in) {  // for the slots in order
    const uint32_t k = in ? key_at(i) : 0u;
    const unsigned tie = __ballot_sync(0xffffffffu, in && k == key);
    const int r = at + __popc(tie & ((1u << lane) - 1));
    at += __popc(tie);
    return in && (k > key || (k == key && r < stay_ties));
  };
  int holes = 0, movers = 0;
  each([&](int i, bool in) {
    const bool stays = stays_at(i, in);
    holes += __popc(__ballot_sync(0xffffffffu, in && !stays && s0 + i < keep));
    movers += __popc(__ballot_sync(0xffffffffu, stays && s0 + i >= keep));
  });
  int hole0, mover0;
  const int all_movers = cluster_sum(lane == 0 ? movers : 0, 2, mover0);
  cluster_sum(lane == 0 ? holes : 0, 3, hole0);
  hole0 += warps_before(holes), mover0 += warps_before(movers);
  at = tie0;
  each([&](int i, bool in) {
    const bool stays = stays_at(i, in);
    const int s = s0 + i;
    const bool hole = in && !stays && s < keep, mover = stays && s >= keep;
    const unsigned h = __ballot_sync(0xffffffffu, hole), m = __ballot_sync(0xffffffffu, mover), below = (1u << lane) - 1;
    if (hole) A.dst[int64_t(b) * A.cap + hole0 + __popc(h & below)] = s;
    if (mover) A.src[int64_t(b) * A.cap + mover0 + __popc(m & below)] = s;
    hole0 += __popc(h), mover0 += __popc(m);
  });
  cluster.sync();  // no block leaves while another may read its shared memory; and the lengths are read
  if (rank == 0 && tid == 0) A.count[b] = all_movers, A.lengths_out[b] = keep;
}

// a warp `rows` movers at a time
__global__ void __launch_bounds__(MOVE_WARPS * 32) move_kernel(const Args A) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  pdl_wait();
  const int count = A.count[b];
  const Pages& P = A.pages;
  const int mask = (1 << P.shift) - 1, words = A.heads * A.row16;
  const int warps = gridDim.x * MOVE_WARPS, warp = blockIdx.x * MOVE_WARPS + (threadIdx.x >> 5);
  const int rows = min(32, max(1, (count + warps - 1) / warps));
  for (int i0 = warp * rows; i0 < count; i0 += warps * rows) {
    const int m = min(rows, count - i0);
    int s = 0, d = 0, ps = -1, pd = -1;
    if (lane < m) {
      s = A.src[int64_t(b) * A.cap + i0 + lane], d = A.dst[int64_t(b) * A.cap + i0 + lane];
      ps = page_of(P, b, s, A.err), pd = page_of(P, b, d, A.err);
      A.weight_out[b * A.weight_out_row + d] = A.weight[b * A.weight_row + s];
      A.position_out[b * A.position_out_row + d] = A.position[b * A.position_row + s];
    }
    for (int r = 0; r < m; ++r) {
      const int rs = __shfl_sync(0xffffffffu, s, r), rd = __shfl_sync(0xffffffffu, d, r);
      const int rps = __shfl_sync(0xffffffffu, ps, r), rpd = __shfl_sync(0xffffffffu, pd, r);
      if (rps < 0 || rpd < 0) continue;
      const char* ks = P.k + rps * P.k_page + (rs & mask) * P.k_token;
      const char* vs = P.v + rps * P.v_page + (rs & mask) * P.v_token;
      char* kd = const_cast<char*>(P.k) + rpd * P.k_page + (rd & mask) * P.k_token;
      char* vd = const_cast<char*>(P.v) + rpd * P.v_page + (rd & mask) * P.v_token;
      for (int j0 = lane; j0 < words; j0 += 64) {  // two words of keys and two of values
        uint4 kx[2], vx[2];
        int64_t ko[2], vo[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = j0 + 32 * e;
          if (j < words) {
            const int h = A.heads > 1 ? j / A.row16 : 0, x = 16 * (j - h * A.row16);
            ko[e] = h * P.k_head + x, vo[e] = h * P.v_head + x;
            kx[e] = *reinterpret_cast<const uint4*>(ks + ko[e]);
            vx[e] = *reinterpret_cast<const uint4*>(vs + vo[e]);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (j0 + 32 * e < words) {
            *reinterpret_cast<uint4*>(kd + ko[e]) = kx[e];
            *reinterpret_cast<uint4*>(vd + vo[e]) = vx[e];
          }
      }
    }
  }
}

// entries of a sequence's lists: holes lie below `keep`, movers at or past it
inline int64_t list_cap(const sc_kv_pages& c, int keep) {
  const int64_t slots = int64_t(c.max_pages) * c.page;
  return slots > keep ? std::min<int64_t>(keep, slots - keep) : 0;
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
  A.heads = kv->kv_heads, A.row16 = kv->head_dim / 8;
  if (kv->k_head == kv->head_dim && kv->v_head == kv->head_dim) A.heads = 1, A.row16 *= kv->kv_heads;
  A.weight_out = weight_out, A.weight_out_row = weight_out_row;
  A.position_out = position_out, A.position_out_row = position_out_row;
  A.lengths_out = lengths_out;
  A.count = static_cast<int32_t*>(workspace);
  A.src = A.count + kv->batch;
  A.dst = A.src + int64_t(kv->batch) * A.cap;
  A.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t slots = int64_t(kv->max_pages) * kv->page;
  int cluster = 1;
  while (cluster < ev::MAX_CLUSTER && slots > int64_t(cluster) * ev::PER_BLOCK) cluster *= 2;
  const int64_t hold = ceil_div(ceil_div(slots, cluster), ev::THREADS) * ev::THREADS;
  const bool held = hold <= ev::MOST;
  const int smem = held ? int(hold) * 4 : 0;
  const auto plan = held ? ev::plan_kernel<true> : ev::plan_kernel<false>;
  // beside the kernel's 17 KB of static shared memory, past 31 KB the dynamic part has to be asked for
  const int asked = smem > 30 * 1024 ? std::max(smem, 48 * 1024 + 16) : 0;
  if (int rc = raise_smem(reinterpret_cast<const void*>(plan), asked, "evict smem attribute")) return rc;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(kv->batch) * cluster);
  cfg.blockDim = dim3(ev::THREADS);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, plan, A)) return cuda_failed(e, "evict plan launch");
  if (A.cap) {
    // four waves of blocks over the batch at most, so that a warp has rows to fetch together
    const int64_t most = std::max<int64_t>(1, ceil_div(4 * 148 * 8, kv->batch));
    cfg.gridDim = dim3(unsigned(std::min<int64_t>(ceil_div(A.cap, ev::MOVE_WARPS), most)), unsigned(kv->batch));
    cfg.blockDim = dim3(ev::MOVE_WARPS * 32);
    cfg.dynamicSmemBytes = 0;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, ev::move_kernel, A)) return cuda_failed(e, "evict move launch");
  }
  return SC_OK;
}
