// Eviction from a paged cache by accumulated attention weight (sc_evict).
//
//   plan_kernel  a cluster of blocks a sequence, each with a stretch of its slots. A slot's key is its weight as an
//                unsigned integer of the same order, the largest integer where its place keeps it; keys stay in shared
//                memory. The key of the last slot that stays is found digit by digit below the bits that all keys
//                share: a histogram of 512 digits a round in every block, summed over the cluster through distributed
//                shared memory, until so few keys are left that they are ranked one against another. Then each warp
//                counts and lists, in slot order, the holes (evicted slots below the budget) and the movers (kept
//                slots past it): as many of one as of the other. Latency bounds it: a round is two barriers and a
//                walk over the histogram (8 sequences of 131072 slots 25 us; with histograms of 2048 digits, of which
//                every block reads 8 KB of each other's, 36).
//   move_kernel  mover i's keys, values, weight and position into hole i. Sources lie at or past the budget and
//                destinations below it, so no row is read that another warp writes, and the order is free. Bandwidth
//                bounds it: a warp fetches the list entries and page ids of its rows at once and keeps four 16-byte
//                words a lane in flight (8 sequences of 131072 slots to 32768: 132 us, the measured copy's rate).
#include <cooperative_groups.h>

#include <algorithm>

#include "pages.cuh"

namespace sc {
namespace ev {

namespace cg = cooperative_groups;

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int BITS = 9, BINS = 1 << BITS;  // a digit a thread
constexpr int FEW = 256;          // keys that are ranked one against another
constexpr int MAX_CLUSTER = 8;
constexpr int STRETCH = 128 * WARPS;  // a block's slots are a multiple
constexpr int MOST = 50 * 1024;   // slots a block can hold the keys of (200 KB); past 8 such blocks keys are made anew
constexpr int OWN = 7 * 1024;     // bytes of plan_kernel's other shared arrays, at most
static_assert(OWN + 4 * MOST <= 227 * 1024, "shared memory of a block");
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
  extern __shared__ __align__(16) uint32_t s_key[];
  __shared__ __align__(16) int s_hist[2][BINS];
  __shared__ int s_warp[4][WARPS], s_pick[3], s_n;
  __shared__ uint32_t s_few[2][FEW];  // this block's, and the cluster's
  __shared__ int4 s_mine[3], s_all[2];  // what the other blocks read; sums over the cluster
  static_assert(sizeof(s_hist) + sizeof(s_warp) + sizeof(s_pick) + sizeof(s_n) + sizeof(s_few) + sizeof(s_mine) +
                    sizeof(s_all) + 64 <= OWN, "and the places' alignment");
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int b = blockIdx.x / blocks, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  const int n = length_of(A.pages, b, A.err), keep = A.keep;
  const float* w = A.weight + b * A.weight_row;
  const int32_t* pos = A.position + b * A.position_row;
  float* wo = A.weight_out + b * A.weight_out_row;
  int32_t* po = A.position_out + b * A.position_out_row;
  // this block's slots, a whole number of steps of 128 to each warp
  const int per = ((n + blocks - 1) / blocks + STRETCH - 1) / STRETCH * STRETCH;
  const int s0 = min(n, rank * per), mine = min(n, s0 + per) - s0;
  auto sync = [&] {
    if (blocks > 1) cluster.sync();
    else __syncthreads();
  };
  const int64_t from = int64_t(A.seen[b]) - A.recent;
  auto is_safe = [&](int32_t p) { return p < A.sinks || p >= from; };
  for (int i = tid; i < 2 * BINS; i += THREADS) s_hist[0][i] = 0;
  // ---- weights and positions, FETCH a thread at a time; those below the budget are copied at once (the evicted among
  // them are overwritten when their slots are filled). Keys; how many slots are kept by their place, and the least and
  // largest of the other keys.
  int safes = 0;
  uint32_t lo = KEPT, hi = 0;
#pragma unroll 1
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
        const bool safe = is_safe(p[u]);
        const uint32_t k = safe ? KEPT : order_of(x[u]);
        safes += safe;
        if (!safe) lo = min(lo, k), hi = max(hi, k);
        if constexpr (HELD) s_key[i] = k;
      }
    }
  }
  if (n <= keep) {
    sync();  // lengths_out may be the lengths themselves
    if (rank == 0 && tid == 0) A.count[b] = 0, A.lengths_out[b] = n;
    return;
  }
  if constexpr (HELD) {  // a step's end holds no slot's key
    const int end = (mine + 127) / 128 * 128;
    for (int i = mine + tid; i < end; i += THREADS) s_key[i] = 0;
  }
  safes = __reduce_add_sync(0xffffffffu, safes);
  lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) s_warp[0][warp] = safes, s_warp[1][warp] = int(lo), s_warp[2][warp] = int(hi);
  __syncthreads();
  if (warp == 0) {
    const bool in = lane < WARPS;
    const int4 v = make_int4(__reduce_add_sync(0xffffffffu, in ? s_warp[0][lane] : 0),
                             int(__reduce_min_sync(0xffffffffu, in ? uint32_t(s_warp[1][lane]) : KEPT)),
                             int(__reduce_max_sync(0xffffffffu, in ? uint32_t(s_warp[2][lane]) : 0u)), 0);
    if (lane == 0) s_mine[0] = v;
  }
  sync();
  if (warp == 0) {
    const int4 v = lane < blocks ? *cluster.map_shared_rank(&s_mine[0], lane) : make_int4(0, int(KEPT), 0, 0);
    const int4 r = make_int4(__reduce_add_sync(0xffffffffu, v.x), int(__reduce_min_sync(0xffffffffu, uint32_t(v.y))),
                             int(__reduce_max_sync(0xffffffffu, uint32_t(v.z))), 0);
    if (lane == 0) s_all[0] = r;
  }
  __syncthreads();
  safes = s_all[0].x, lo = uint32_t(s_all[0].y), hi = uint32_t(s_all[0].z);
  // more kept places than slots stay (positions that repeat): only they are ranked, by weight
  const bool crowded = safes > keep;
  auto make = [&](int i) -> uint32_t {
    const bool safe = is_safe(pos[s0 + i]);
    return crowded ? (safe ? order_of(w[s0 + i]) : 0u) : safe ? KEPT : order_of(w[s0 + i]);
  };
  if (crowded) {
    lo = 0, hi = KEPT - 1;
    if constexpr (HELD) {
      for (int i = tid; i < mine; i += THREADS) s_key[i] = make(i);
      __syncthreads();
    }
  }
  auto key_at = [&](int i) { return HELD ? s_key[i] : make(i); };
  // ---- the key of the last slot that stays: slots above it stay, `want` of those at it
  int want = crowded ? keep : keep - safes;
  uint32_t key = KEPT;
  if (want > 0) {
    int bits = hi > lo ? 32 - __clz(hi ^ lo) : 0;  // those that the keys below KEPT do not share
    key = bits < 32 ? (hi >> bits) << bits : 0u;
    int left = INT32_MAX;  // keys that begin as `key` does
    for (int round = 0; bits > 0 && left > FEW; ++round) {
      const int take = min(bits, BITS), shift = bits - take;
      const uint32_t known = bits < 32 ? ~0u << bits : 0u, digit = (1u << take) - 1;
      int* hist = s_hist[round & 1];
#pragma unroll 4
      for (int i = tid; i < mine; i += THREADS) {
        const uint32_t k = key_at(i);
        if (k != KEPT && (k & known) == key) atomicAdd(&hist[(k >> shift) & digit], 1);
      }
      sync();
      // a digit a thread, from the top down
      const int d = BINS - 1 - tid;
      int v = 0;
#pragma unroll
      for (int r = 0; r < MAX_CLUSTER; ++r)
        if (r < blocks) v += *cluster.map_shared_rank(hist + d, r);
      s_hist[(round + 1) & 1][d] = 0;  // which no block reads any more: the next round's
      const int inc = warp_scan(v);
      if (lane == 31) s_warp[0][warp] = inc;
      __syncthreads();
      int upto = inc - v;
#pragma unroll
      for (int q = 0; q < WARPS; ++q) upto += q < warp ? s_warp[0][q] : 0;
      if (upto < want && want <= upto + v) s_pick[0] = d, s_pick[1] = upto, s_pick[2] = v;
      __syncthreads();
      key |= uint32_t(s_pick[0]) << shift;
      want -= s_pick[1];
      left = s_pick[2];
      bits = shift;
    }
    if (bits > 0) {  // few keys are left: each counts those above it
      const uint32_t known = ~0u << bits;
      if (tid == 0) s_n = 0;
      __syncthreads();
#pragma unroll 4
      for (int i = tid; i < mine; i += THREADS) {
        const uint32_t k = key_at(i);
        if (k != KEPT && (k & known) == key) s_few[0][atomicAdd(&s_n, 1)] = k;
      }
      sync();
      if (warp < blocks) {
        int at = 0, m = 0;
        for (int r = 0; r <= warp; ++r) at += m, m = *cluster.map_shared_rank(&s_n, r);
        const uint32_t* from = cluster.map_shared_rank(&s_few[0][0], warp);
        for (int i = lane; i < m; i += 32) s_few[1][at + i] = from[i];
      }
      __syncthreads();
      if (tid < left) {
        const uint32_t k = s_few[1][tid];
        int above = 0, equal = 0;
        for (int i = 0; i < left; ++i) above += s_few[1][i] > k, equal += s_few[1][i] == k;
        if (above < want && want <= above + equal) s_pick[0] = int(k), s_pick[1] = above;  // equal keys write alike
      }
      __syncthreads();
      key = uint32_t(s_pick[0]);
      want -= s_pick[1];
    }
  }
  // ---- the lists, in slot order: warp w has a stretch of this block's slots, a lane four of them at a step
  const int span = per / WARPS, w0 = warp * span, w1 = min(mine, w0 + span);
  auto keys_at = [&](int i) -> uint4 {  // zeros past the end
    if constexpr (HELD) {
      uint4 k = *reinterpret_cast<const uint4*>(s_key + i);
      return k;
    } else {
      return make_uint4(i < mine ? make(i) : 0u, i + 1 < mine ? make(i + 1) : 0u, i + 2 < mine ? make(i + 2) : 0u,
                        i + 3 < mine ? make(i + 3) : 0u);
    }
  };
  // per warp: its slots at `key`, those of them below the budget, and the holes and movers without them
  int ties = 0, low = 0, holes = 0, movers = 0;
  for (int i0 = w0; i0 < w1; i0 += 128) {
    const uint4 k4 = keys_at(i0 + 4 * lane);
    const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + 4 * lane + e;
      if (i < w1) {
        const bool below = s0 + i < keep;
        ties += k[e] == key, low += below && k[e] == key;
        holes += below && k[e] < key, movers += !below && k[e] > key;
      }
    }
  }
  ties = __reduce_add_sync(0xffffffffu, ties), low = __reduce_add_sync(0xffffffffu, low);
  holes = __reduce_add_sync(0xffffffffu, holes), movers = __reduce_add_sync(0xffffffffu, movers);
  // what the warps and blocks before this one have of x and y; the whole cluster's in s_all
  auto before = [&](int use, int x, int y) -> int2 {
    if (lane == 0) s_warp[1][warp] = x, s_warp[2][warp] = y;
    __syncthreads();
    if (warp == 0) {
      const int xs = lane < WARPS ? s_warp[1][lane] : 0, ys = lane < WARPS ? s_warp[2][lane] : 0;
      const int xi = warp_scan(xs), yi = warp_scan(ys);
      if (lane < WARPS) s_warp[1][lane] = xi - xs, s_warp[2][lane] = yi - ys;
      if (lane == 31) s_mine[use] = make_int4(xi, yi, 0, 0);
    }
    sync();
    if (warp == 0) {
      const int4 v = lane < blocks ? *cluster.map_shared_rank(&s_mine[use], lane) : make_int4(0, 0, 0, 0);
      const int4 r = make_int4(__reduce_add_sync(0xffffffffu, v.x), __reduce_add_sync(0xffffffffu, v.y),
                               __reduce_add_sync(0xffffffffu, lane < rank ? v.x : 0),
                               __reduce_add_sync(0xffffffffu, lane < rank ? v.y : 0));
      if (lane == 0) s_all[1] = r;
    }
    __syncthreads();
    const int2 r = make_int2(s_warp[1][warp] + s_all[1].z, s_warp[2][warp] + s_all[1].w);
    return r;
  };
  // of the slots at `key` the lowest `stay` stay; in slot order, so a warp's below the budget before its others
  int tie = before(1, ties, 0).x;
  const int stay = key == KEPT ? s_all[1].x : want;
  const int here = min(max(stay - tie, 0), ties), here_low = min(here, low);
  __syncthreads();  // s_all has been read
  const int2 at = before(2, holes + low - here_low, movers + here - here_low);
  const int all_movers = s_all[1].y;
  int32_t* dst = A.dst + int64_t(b) * A.cap + at.x;
  int32_t* src = A.src + int64_t(b) * A.cap + at.y;
  for (int i0 = w0; i0 < w1; i0 += 128) {
    const uint4 k4 = keys_at(i0 + 4 * lane);
    const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
    unsigned stays = 0, equal = 0, in = 0, below = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + 4 * lane + e;
      stays |= unsigned(k[e] > key) << e, equal |= unsigned(k[e] == key) << e;
      in |= unsigned(i < w1) << e, below |= unsigned(s0 + i < keep) << e;
    }
    equal &= in;
    if (here == ties) {
      stays |= equal;
    } else if (here > 0) {  // one warp of the cluster
      const int c = __popc(equal), inc = warp_scan(c);
      int r = tie + inc - c;
      tie += __shfl_sync(0xffffffffu, inc, 31);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((equal >> e) & 1) stays |= unsigned(r++ < stay) << e;
    }
    const unsigned h = in & below & ~stays, m = in & ~below & stays;
    const int c = __popc(h) | __popc(m) << 16, inc = warp_scan(c), ex = inc - c, sum = __shfl_sync(0xffffffffu, inc, 31);
    int32_t *hp = dst + (ex & 0xffff), *mp = src + (ex >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if ((h >> e) & 1) *hp++ = s0 + i0 + 4 * lane + e;
      if ((m >> e) & 1) *mp++ = s0 + i0 + 4 * lane + e;
    }
    dst += sum & 0xffff, src += sum >> 16;
  }
  sync();  // no block leaves while another may read its shared memory; and the lengths are read
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
  // One block up to two stretches of slots, where a cluster's barriers cost more than they share out (one sequence of
  // 2304: 10.4 us, with two blocks 11.5; 64 of 4096: 32.9 and 34.0); past that a stretch a block (one of 8192: four
  // blocks 14.4, one 16.5, eight 14.6; four of 32768: eight 26.1, four 28.7).
  int cluster = 1;
  while (cluster < ev::MAX_CLUSTER && slots > int64_t(cluster > 1 ? cluster : 2) * ev::STRETCH) cluster *= 2;
  const int64_t hold = ceil_div(ceil_div(slots, cluster), ev::STRETCH) * ev::STRETCH;
  const bool held = hold <= ev::MOST;
  const int smem = held ? int(hold) * 4 : 0;
  const auto plan = held ? ev::plan_kernel<true> : ev::plan_kernel<false>;
  // 48 KB with the kernel's own arrays go without asking; raise_smem asks for more than that only
  const int asked = smem + ev::OWN > 48 * 1024 ? std::max(smem, 48 * 1024 + 16) : 0;
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
