// Attention of one new token a sequence over a batch's paged cache, the weights accumulated on request
// (sc_decode_attention): o = sum_s p_s v_s, p = softmax_s(scale q . k_s). Every key and value is read once, so the
// cache's bytes bound it; what the kernel has to do is keep enough of them in flight.
//
//   attend_kernel  The batch's caches are cut into units of 64 slots or more (a tile a warp), counted over sequence,
//                  key/value head and slot, and every block takes an equal run of units: ragged lengths balance, and
//                  a long cache spreads over all SMs. A block joins its warps' results in shared memory; a run that
//                  covers a head's whole length writes the output, the others partial results (at most two a block).
//   join_kernel    joins the partial results in block order (the same bits on every run), and adds the weights.
//   starts_kernel  first, for more than two sequences for each thread of an attending block: how many units lie before
//                  each. (Up to as many, every block counts them itself: 129 of up to 512 tokens 28 us, with this kernel
//                  32. Past it that took passes in every block of both kernels: 4096 rows of up to 512 tokens, 16 / 2
//                  heads of 256, 1080 us, with this kernel 778; 65535 of up to 64, heads of 64, 134 ms and 3.8.)
//
// A warp's tile goes from memory straight into tensor-core fragments (mma.sync m16n8k16; up to eight query heads share
// the key/value head, so a product of 16 slots by 8 heads has little padding, and 128-row tcgen05 products would
// have nothing to fill them). The order of a sum's terms is free, so each lane takes 16-byte pieces of rows:
//   scores   S^T = K Q^T, 16 slots by 8 heads: lane (g, t) holds dims 8 (4 j + t) .. + 7 of slots g and g + 8, four
//            dims to a product; Q is laid out the same way;
//   values   O^T = V^T P^T, 16 dims by 8 heads: the lane holds dims 64 i + 8 g .. + 7 of slots 2t, 2t + 1, 2t + 8 and
//            2t + 9, paired by byte permutes; the scores' accumulators become P^T's fragments by movmatrix.
// The softmax is online: scores are taken relative to a running maximum a head, moved only when a score passes it by
// 2^8 (a vote a tile instead of a reduction; float32 holds the larger probabilities as exactly). A probability enters
// the value product as two terms of the activations' type (its rounding and the rest), so that only the output is
// rounded to 16 bits: to 2^-16 of itself in bfloat16, whose exponents reach down to float32's. Float16's end at 2^-24, so
// there the maximum moves with every larger score and stands at 2^15: a probability is within 2^-22 of itself, and where
// its terms run out of bits within 2^-40 of the largest (with the peak at 1 a tail of slots below 2^-25 behind it was
// missing from the output). The next tile's keys load while this tile's softmax and value product run, its values after.
// Measured: 8 sequences of 131072 tokens, 16 / 2 heads of 256, 325 to 330 us (6.5 TB/s, what a copy reaches); one of 8192
// 11.8 us, of which the bytes are 2.6: the launch, one or two tiles a warp, the join. 32 ragged sequences to 9001, 32 / 8
// heads of 128: 115 us (5.6 TB/s), with the weights gathered 125 (the scores' write and the join's read of them). Heads of
// 256 take all 255 registers and spill 84 bytes of stores and 124 of loads a thread.
#include <algorithm>
#include <type_traits>

#include "mma_decode.cuh"
#include "pages.cuh"

namespace sc {
namespace da {

constexpr int HEADS = 8;       // query heads of a block: the products' N
// Warps of a block and blocks of an SM, as many as the registers of a warp's tile leave room for. Heads of 256: one
// block, as two of half as many warps write twice the partial results (one sequence of 8192: 16.1 us against 12.6).
// Smaller heads: three, as fewer and larger ones leave more of the memory idle where runs end and start (a ragged batch:
// 148 us with one block of 12 warps, 132 with two of 6 or three of 4; short sequences 10.0, 8.4 and 8.0).
constexpr int warps_of(int dp) { return dp == 256 ? 8 : 4; }
constexpr int blocks_per_sm(int dp) { return dp == 256 ? 1 : 3; }
constexpr int SMS = 148;
// log2 by which a score may pass the running maximum, and of what a probability at the maximum is taken as
template <typename T> constexpr float SLACK = std::is_same_v<T, __half> ? 0.f : 8.f;
template <typename T> constexpr float TOP = std::is_same_v<T, __half> ? 15.f : 0.f;
constexpr int JOIN_THREADS = 256;

struct Args {
  Pages pages;
  const void* q;
  int64_t q_row, q_head;
  int batch, q_heads, kv_heads, group, head_tiles, dim, columns;  // columns: blocks that share the units
  float scale_log2;
  void* out;
  float* weight;
  int64_t weight_row;
  float* scores;      // (batch, kv_heads, head_tiles, slots, pack) with weights, log2 domain
  int64_t slots;
  int pack;           // heads a slot's scores are stored for: min(group, 8) rounded up to a power of two
  float* part_o;      // (head_tiles, columns, 2, 8, DP) unnormalized outputs of runs that cover part of a head
  float2* part_ml;    // (head_tiles, columns, 2, 8) their maxima and sums
  float2* whole_ml;   // (batch, q_heads) those of heads that one block covered
  int32_t* starts;    // (batch + 1) units before each sequence, a head's, and in all; NULL where the blocks count
  int* err;
};

__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
// 2^x to 2^-22 of it, zero below 2^-126: a probability relative to a running maximum
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.f : m; }

template <int N>
__device__ __forceinline__ int block_sum(int v, int* sh) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int i = 0; i < N / 32; ++i) t += sh[i];
  __syncthreads();
  return t;
}
template <int N>
__device__ __forceinline__ int block_scan(int v, int* sh, int& total) {  // inclusive
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) sh[warp] = v;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < N / 32; ++w) {
    if (w < warp) v += sh[w];
    total += sh[w];
  }
  __syncthreads();
  return v;
}

// The units' numbering: sequence after sequence, in each head after head. X blocks (at most as many as there are
// units, so that each has one) share U units as evenly as whole ones go: the first U % X blocks take one more.
struct Split {
  uint32_t each, more;  // U / X, U % X
  __device__ __forceinline__ Split(uint32_t U, uint32_t X) : each(U / X), more(U % X) {}
  __device__ __forceinline__ uint32_t start(uint32_t x) const { return x * each + min(x, more); }
  __device__ __forceinline__ uint32_t block_of(uint32_t u) const {
    const uint32_t longer = more * (each + 1);
    return u < longer ? u / (each + 1) : more + (u - longer) / each;
  }
};

template <typename T, int DP, int SUB>
__global__ void __launch_bounds__(warps_of(DP) * 32, blocks_per_sm(DP)) attend_kernel(const Args A) {
  constexpr int WARPS = warps_of(DP), THREADS = WARPS * 32;
  constexpr int KC = DP / 32, VC = DP / 64, TILE = 16 * SUB, UNIT = WARPS * TILE;
  constexpr int IDS = (TILE + 31) / 32;
  __shared__ uint4 s_q[KC][32];
  extern __shared__ __align__(16) float s_dyn[];
  auto s_o = reinterpret_cast<float (*)[HEADS][DP]>(s_dyn);  // [WARPS]
  __shared__ float s_m[WARPS][HEADS], s_l[WARPS][HEADS];
  __shared__ int s_sum[WARPS], s_before, s_b;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int ht = blockIdx.y;
  const uint32_t x = blockIdx.x;
  if (A.starts) pdl_wait();
  pdl_launch_dependents();
  // the units in all, and the sequence that holds this block's first one
  int U, to = 0;
  int n0 = 0, n1 = 0;  // of two sequences a thread
  if (!A.starts && 2 * tid < A.batch) {
    n0 = (length_of(A.pages, 2 * tid, A.err) + UNIT - 1) / UNIT;
    if (2 * tid + 1 < A.batch) n1 = (length_of(A.pages, 2 * tid + 1, A.err) + UNIT - 1) / UNIT;
  }
  if (A.starts) U = A.starts[A.batch];
  else if (A.batch == 1) U = (length_of(A.pages, 0, nullptr) + UNIT - 1) / UNIT;
  else to = block_scan<THREADS>(n0 + n1, s_sum, U);
  U *= A.kv_heads;
  const uint32_t X = min(A.columns, U);
  if (x >= X) return;
  const Split split(U, X);
  int u = split.start(x);
  const int u1 = split.start(x + 1);
  int b = 0, before = 0;
  if (A.starts) {  // the last sequence that begins at or before it: 32 places at a time, every warp for itself
    const int w = u / A.kv_heads;
#pragma unroll 1
    for (int end = A.batch; end - b > 1;) {
      const int step = (end - b + 31) / 32, at = b + lane * step;
      const int n = __popc(__ballot_sync(0xffffffffu, at < end && A.starts[at] <= w));
      b += max(n - 1, 0) * step;
      end = min(end, b + step);
    }
    before = A.starts[b];
  } else if (A.batch > 1) {
    if (tid == 0) s_b = -1;
    __syncthreads();
    if (u >= (to - n1 - n0) * A.kv_heads && u < to * A.kv_heads) {
      const bool second = u >= (to - n1) * A.kv_heads;
      s_b = 2 * tid + second, s_before = to - n1 - (second ? 0 : n0);
    }
    __syncthreads();
    b = s_b, before = s_before;
    if (b < 0) return;  // the lengths changed under the kernel
  }
  int hk, ul;
  {
    const int n = (length_of(A.pages, b, nullptr) + UNIT - 1) / UNIT;
    if (n == 0) return;  // as above
    const uint32_t in = u - before * A.kv_heads;
    hk = in / n, ul = in % n;
  }
  const Pages& P = A.pages;
  const int mask = (1 << P.shift) - 1, chunks = A.dim / 8;
  const int heads = min(HEADS, A.group - ht * HEADS);  // of this block
  while (u < u1 && b < A.batch) {
    const int len = length_of(P, b, nullptr), n_units = (len + UNIT - 1) / UNIT;
    if (n_units == 0 || hk == A.kv_heads) {
      ++b, hk = 0, ul = 0;
      continue;
    }
    const int ue = min(n_units, ul + (u1 - u));
    // ---- this warp's tiles
    const int end = min(len, ue * UNIT);
    int base = (ul * WARPS + warp) * TILE;
    const char* kb = P.k + hk * P.k_head + 16 * t;
    const char* vb = P.v + hk * P.v_head + 16 * g;
    const int32_t* table = P.table + b * P.table_row;
    // page ids of a tile's slots, lane l that of slots l and l + 32; -1 past the end or outside the pool
    auto load_ids = [&](int at, int (&id)[IDS]) {
#pragma unroll
      for (int i = 0; i < IDS; ++i) {
        const int s = at + lane + 32 * i;
        id[i] = -1;
        if (s < end && lane + 32 * i < TILE) {
          id[i] = __ldg(table + (s >> P.shift));
          if (unsigned(id[i]) >= unsigned(P.pool_pages)) {
            record_error(A.err, SC_ERR_PAGE);
            id[i] = -1;
          }
        }
      }
    };
    uint4 kf[SUB][2][KC], vf[SUB][4][VC];
    auto load_k = [&](int at, const int (&id)[IDS]) -> uint32_t {  // returns which of the lane's slots hold a token
      uint32_t valid = 0;
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int o = 16 * s + 8 * r + g, page = __shfl_sync(0xffffffffu, id[s / 2], o & 31);
          const char* p = kb + page * P.k_page + ((at + o) & mask) * P.k_token;
          if (page >= 0) valid |= 1u << (2 * s + r);
#pragma unroll
          for (int j = 0; j < KC; ++j) {
            kf[s][r][j] = make_uint4(0, 0, 0, 0);
            if (page >= 0 && 4 * j + t < chunks) kf[s][r][j] = load16(p + 64 * j);
          }
        }
      return valid;
    };
    auto load_v = [&](int at, const int (&id)[IDS]) {
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int o = 16 * s + 8 * (r >> 1) + 2 * t + (r & 1), page = __shfl_sync(0xffffffffu, id[s / 2], o & 31);
          const char* p = vb + page * P.v_page + ((at + o) & mask) * P.v_token;
#pragma unroll
          for (int i = 0; i < VC; ++i) {
            vf[s][r][i] = make_uint4(0, 0, 0, 0);
            if (page >= 0 && 8 * i + g < chunks) vf[s][r][i] = load16(p + 128 * i);
          }
        }
    };
    float o[VC][4][4];
#pragma unroll
    for (int i = 0; i < VC; ++i)
#pragma unroll
      for (int m = 0; m < 4; ++m) o[i][m][0] = o[i][m][1] = o[i][m][2] = o[i][m][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, b0 = 0.f, b1 = 0.f, l0 = 0.f, l1 = 0.f;  // of heads 2t and 2t + 1
    int id[IDS], next[IDS];
    load_ids(base, id);
    // the heads' queries, in the products' order
#pragma unroll 1
    for (int i = tid; i < KC * 32; i += THREADS) {
      const int c = (i / 32) * 4 + (i & 3), h = (i & 31) >> 2;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (h < heads && c < chunks)
        v = *reinterpret_cast<const uint4*>(static_cast<const T*>(A.q) + b * A.q_row +
                                            int64_t(hk * A.group + ht * HEADS + h) * A.q_head + 8 * c);
      s_q[i / 32][i & 31] = v;
    }
    uint32_t valid = load_k(base, id);
    load_v(base, id);
    load_ids(base + UNIT, next);
    __syncthreads();
#pragma unroll 1
    for (; base < end; base += UNIT) {
      float s[SUB][4], s2[SUB][4];  // two chains of products
#pragma unroll
      for (int i = 0; i < SUB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = s2[i][e] = 0.f;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const uint4 q = s_q[j][lane];
#pragma unroll
        for (int i = 0; i < SUB; ++i) {
          const uint4 &ka = kf[i][0][j], &kc = kf[i][1][j];
          const uint32_t a0[4] = {ka.x, kc.x, ka.y, kc.y}, a1[4] = {ka.z, kc.z, ka.w, kc.w};
          mma16816<T>(s[i], a0, q.x, q.y);
          mma16816<T>(s2[i], a1, q.z, q.w);
        }
      }
      const uint32_t in = valid;
      valid = load_k(base + UNIT, next);
      float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool ok = (in >> (2 * i + r)) & 1;
          s[i][2 * r] = ok ? (s[i][2 * r] + s2[i][2 * r]) * A.scale_log2 : -INFINITY;
          s[i][2 * r + 1] = ok ? (s[i][2 * r + 1] + s2[i][2 * r + 1]) * A.scale_log2 : -INFINITY;
          x0 = fmaxf(x0, s[i][2 * r]);
          x1 = fmaxf(x1, s[i][2 * r + 1]);
        }
      }
      if (A.scores) {
#pragma unroll
        for (int i = 0; i < SUB; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int slot = base + 16 * i + 8 * r + g;
            if (slot < end && 2 * t < A.pack) {
              float* to = A.scores + (((int64_t(b) * A.kv_heads + hk) * A.head_tiles + ht) * A.slots + slot) * A.pack + 2 * t;
              if (A.pack > 1) *reinterpret_cast<float2*>(to) = make_float2(s[i][2 * r], s[i][2 * r + 1]);
              else *to = s[i][2 * r];
            }
          }
      }
      if (__any_sync(0xffffffffu, x0 > m0 + SLACK<T> || x1 > m1 + SLACK<T>)) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, w));
          x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, w));
        }
        x0 = fmaxf(x0, m0), x1 = fmaxf(x1, m1);
        b0 = finite_or_0(x0), b1 = finite_or_0(x1);
        const float c0 = ex2(m0 - b0), c1 = ex2(m1 - b1);
        b0 -= TOP<T>, b1 -= TOP<T>;
        m0 = x0, m1 = x1;
        l0 *= c0, l1 *= c1;
#pragma unroll
        for (int i = 0; i < VC; ++i)
#pragma unroll
          for (int m = 0; m < 4; ++m) o[i][m][0] *= c0, o[i][m][1] *= c1, o[i][m][2] *= c0, o[i][m][3] *= c1;
      }
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float p0 = ex2(s[i][2 * r] - b0), p1 = ex2(s[i][2 * r + 1] - b1);
          l0 += p0, l1 += p1;
          const uint32_t h = pack2<T>(p0, p1);
          const float2 back = unpack2<T>(h);
          hi[r] = transpose8x8(h);
          lo[r] = transpose8x8(pack2<T>(p0 - back.x, p1 - back.y));
        }
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          const uint32_t* r0 = reinterpret_cast<const uint32_t*>(&vf[i][0][c]);
          const uint32_t* r1 = reinterpret_cast<const uint32_t*>(&vf[i][1][c]);
          const uint32_t* r2 = reinterpret_cast<const uint32_t*>(&vf[i][2][c]);
          const uint32_t* r3 = reinterpret_cast<const uint32_t*>(&vf[i][3][c]);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const uint32_t a[4] = {__byte_perm(r0[m], r1[m], 0x5410), __byte_perm(r0[m], r1[m], 0x7632),
                                   __byte_perm(r2[m], r3[m], 0x5410), __byte_perm(r2[m], r3[m], 0x7632)};
            mma16816<T>(o[c][m], a, hi[0], hi[1]);
            mma16816<T>(o[c][m], a, lo[0], lo[1]);
          }
        }
      }
      load_v(base + UNIT, next);
      load_ids(base + 2 * UNIT, next);
    }
    // ---- the warps' results joined, from here on with a probability at the maximum as 1
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, w);
      l1 += __shfl_xor_sync(0xffffffffu, l1, w);
    }
    constexpr float DOWN = 1.f / float(1 << int(TOP<T>));
    l0 *= DOWN, l1 *= DOWN;
    if (g == 0) s_m[warp][2 * t] = m0, s_m[warp][2 * t + 1] = m1, s_l[warp][2 * t] = l0, s_l[warp][2 * t + 1] = l1;
    __syncthreads();
    float M0 = -INFINITY, M1 = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M0 = fmaxf(M0, s_m[w][2 * t]), M1 = fmaxf(M1, s_m[w][2 * t + 1]);
    const float c0 = DOWN * ex2(m0 - finite_or_0(M0)), c1 = DOWN * ex2(m1 - finite_or_0(M1));
#pragma unroll
    for (int i = 0; i < VC; ++i) {
      float4* to = reinterpret_cast<float4*>(&s_o[warp][2 * t][64 * i + 8 * g]);
      to[0] = make_float4(o[i][0][0] * c0, o[i][0][2] * c0, o[i][1][0] * c0, o[i][1][2] * c0);
      to[1] = make_float4(o[i][2][0] * c0, o[i][2][2] * c0, o[i][3][0] * c0, o[i][3][2] * c0);
      to = reinterpret_cast<float4*>(&s_o[warp][2 * t + 1][64 * i + 8 * g]);
      to[0] = make_float4(o[i][0][1] * c1, o[i][0][3] * c1, o[i][1][1] * c1, o[i][1][3] * c1);
      to[1] = make_float4(o[i][2][1] * c1, o[i][2][3] * c1, o[i][3][1] * c1, o[i][3][3] * c1);
    }
    __syncthreads();
    const bool whole = ul == 0 && ue == n_units;
    const int64_t part = ((int64_t(ht) * A.columns + x) * 2 + (ul == 0)) * HEADS;  // 0: a head's later run, 1: its first
#pragma unroll 1
    for (int e = tid; e < heads * (DP / 4); e += THREADS) {
      const int h = e / (DP / 4), d = 4 * (e % (DP / 4));
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w][h]);
      const float mb = finite_or_0(M);
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        L += s_l[w][h] * ex2(s_m[w][h] - mb);
        const float4 v = *reinterpret_cast<const float4*>(&s_o[w][h][d]);
        r.x += v.x, r.y += v.y, r.z += v.z, r.w += v.w;
      }
      const int64_t row = int64_t(b) * A.q_heads + hk * A.group + ht * HEADS + h;
      if (whole) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        if (d < A.dim)
          *reinterpret_cast<uint2*>(static_cast<T*>(A.out) + row * A.dim + d) =
              make_uint2(pack2<T>(r.x * inv, r.y * inv), pack2<T>(r.z * inv, r.w * inv));
        if (d == 0 && A.scores) A.whole_ml[row] = make_float2(mb, L);
      } else {
        *reinterpret_cast<float4*>(A.part_o + (part + h) * DP + d) = r;
        if (d == 0) A.part_ml[part + h] = make_float2(M, L);
      }
    }
    __syncthreads();  // s_q, s_m and s_o are the next run's
    u += ue - ul;
    ul = 0;
    ++hk;
  }
}

// The blocks that share the units of a sequence's heads: head hk's are first(hk) .. last(hk), none when n is 0.
struct Share {
  Split split;
  int before, n;
  __device__ __forceinline__ int first(int hk) const { return split.block_of(before + hk * n); }
  __device__ __forceinline__ int last(int hk) const { return split.block_of(before + hk * n + n - 1); }
};
template <int N>
__device__ __forceinline__ Share share_of(const Args& A, int unit, int b, int* sh) {
  const int n = (length_of(A.pages, b, nullptr) + unit - 1) / unit;
  int U = n, before = 0;
  if (A.starts) {
    U = A.starts[A.batch], before = A.starts[b];
  } else if (A.batch > 1) {
    int all = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < A.batch; i += N) {
      const int k = (length_of(A.pages, i, nullptr) + unit - 1) / unit;
      all += k;
      if (i < b) before += k;
    }
    U = block_sum<N>(all, sh), before = block_sum<N>(before, sh);
  }
  U = max(1, U * A.kv_heads);  // there may be none
  return {Split(U, min(A.columns, U)), before * A.kv_heads, n};
}

// One block: each thread a run of sequences.
constexpr int STARTS_THREADS = 1024;
__global__ void __launch_bounds__(STARTS_THREADS) starts_kernel(const Args A, int unit) {
  __shared__ int sh[STARTS_THREADS / 32];
  pdl_launch_dependents();
  const int per = (A.batch + STARTS_THREADS - 1) / STARTS_THREADS, b0 = threadIdx.x * per, b1 = min(A.batch, b0 + per);
  int n = 0, total;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) n += (length_of(A.pages, b, A.err) + unit - 1) / unit;
  int at = block_scan<STARTS_THREADS>(n, sh, total) - n;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) {
    A.starts[b] = at;
    at += (length_of(A.pages, b, nullptr) + unit - 1) / unit;
  }
  if (threadIdx.x == 0) A.starts[A.batch] = total;
}

// Blocks 0 .. batch x q_heads - 1: a query head's output from its partial results (zeros for an empty sequence). The
// rest, with weights: JOIN_THREADS slots of a sequence, a thread a slot, PACK scores at a time.
template <typename T, int DP, int PACK>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const Args A, int unit, int slot_blocks) {
  constexpr int LANES = DP / 4, GROUPS = JOIN_THREADS / LANES;  // threads of a row, and rows read side by side
  __shared__ int sh[JOIN_THREADS / 32];
  __shared__ __align__(16) float s_o[GROUPS][DP];
  __shared__ float2 s_gml[GROUPS];
  extern __shared__ float2 s_ml[];  // of every query head (weights)
  const int tid = threadIdx.x;
  const int outs = A.batch * A.q_heads;
  if (int(blockIdx.x) < outs) {
    const int b = blockIdx.x / A.q_heads, h = blockIdx.x % A.q_heads, hk = h / A.group, hh = h % A.group;
    const int ht = hh / HEADS, hr = hh % HEADS;
    T* out = static_cast<T*>(A.out) + int64_t(blockIdx.x) * A.dim;
    const Share s = share_of<JOIN_THREADS>(A, unit, b, sh);
    const int first = s.n ? s.first(hk) : 0, last = s.n ? s.last(hk) : 0;
    pdl_wait();
    if (s.n == 0) {
#pragma unroll 1
      for (int d = tid; d < A.dim; d += JOIN_THREADS) out[d] = from_f32<T>(0.f);
      return;
    }
    if (first == last) return;  // one block covered it
    // each row of threads an online join of every GROUPS-th partial result, four at a time
    const int row = tid / LANES, d = 4 * (tid % LANES);
    const int64_t base = int64_t(ht) * A.columns * 2 * HEADS + hr;
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int x0 = first + row; x0 <= last; x0 += 4 * GROUPS) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int x = x0 + i * GROUPS;
        ml[i] = make_float2(-INFINITY, 0.f);
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (x <= last) {
          const int64_t at = base + (int64_t(x) * 2 + (x == first)) * HEADS;
          ml[i] = A.part_ml[at];
          v[i] = *reinterpret_cast<const float4*>(A.part_o + at * DP + d);
        }
      }
      const float top = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), M), mb = finite_or_0(top);
      const float c = ex2(M - mb);
      M = top;
      L *= c, o.x *= c, o.y *= c, o.z *= c, o.w *= c;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = ex2(ml[i].x - mb);
        L += ml[i].y * e;
        o.x += v[i].x * e, o.y += v[i].y * e, o.z += v[i].z * e, o.w += v[i].w * e;
      }
    }
    *reinterpret_cast<float4*>(&s_o[row][d]) = o;
    if (d == 0) s_gml[row] = make_float2(M, L);
    __syncthreads();
    if (row == 0 && d < A.dim) {
#pragma unroll
      for (int i = 1; i < GROUPS; ++i) M = fmaxf(M, s_gml[i].x);
      const float mb = finite_or_0(M);
      L = 0.f;
      o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(&s_o[i][d]);
        const float e = ex2(s_gml[i].x - mb);
        L += s_gml[i].y * e;
        o.x += v.x * e, o.y += v.y * e, o.z += v.z * e, o.w += v.w * e;
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      *reinterpret_cast<uint2*>(out + d) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
    }
    return;
  }
  const int e = blockIdx.x - outs, b = e / slot_blocks, s0 = (e % slot_blocks) * JOIN_THREADS, s = s0 + tid;
  const int len = length_of(A.pages, b, nullptr);
  if (s0 >= len) return;
  const Share share = share_of<JOIN_THREADS>(A, unit, b, sh);
  const int tiles = A.kv_heads * A.head_tiles;
  const float* from = A.scores + (int64_t(b) * tiles * A.slots + s) * PACK;
  const bool live = s < len;
  pdl_wait();
  // the scores of the first tiles load while the heads' statistics are worked out
  constexpr int AHEAD = PACK == 8 ? 4 : 8;
  float x[AHEAD][PACK];
  auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float* p = from + int64_t(t0 + i) * A.slots * PACK;
#pragma unroll
      for (int h = 0; h < PACK; ++h) x[i][h] = -INFINITY;
      if (live && t0 + i < tiles) {
        if constexpr (PACK == 1) {
          x[i][0] = *p;
        } else if constexpr (PACK == 2) {
          const float2 v = *reinterpret_cast<const float2*>(p);
          x[i][0] = v.x, x[i][1] = v.y;
        } else {
#pragma unroll
          for (int h = 0; h < PACK; h += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + h);
            x[i][h] = v.x, x[i][h + 1] = v.y, x[i][h + 2] = v.z, x[i][h + 3] = v.w;
          }
        }
      }
    }
  };
  load(0);
  const float old = live ? A.weight[b * A.weight_row + s] : 0.f;
  // s_ml: (tiles, PACK) the heads' maxima and the inverses of their sums, zeros for heads that there are not
#pragma unroll 1
  for (int i = tid; i < tiles * PACK; i += JOIN_THREADS) {
    const int hk = i / PACK / A.head_tiles, ht = i / PACK % A.head_tiles, hh = ht * HEADS + i % PACK;
    float2 ml = make_float2(0.f, 0.f);
    if (hh < A.group) {
      const int first = share.first(hk), last = share.last(hk);
      if (first == last) {
        ml = A.whole_ml[int64_t(b) * A.q_heads + hk * A.group + hh];
      } else {
        const int64_t base = int64_t(ht) * A.columns * 2 * HEADS + i % PACK;
        float M = -INFINITY, L = 0.f;
#pragma unroll 2
        for (int k = first; k <= last; ++k) {
          const float2 v = A.part_ml[base + (int64_t(k) * 2 + (k == first)) * HEADS];
          const float top = fmaxf(M, v.x), mb = finite_or_0(top);
          L = L * ex2(M - mb) + v.y * ex2(v.x - mb);
          M = top;
        }
        ml = make_float2(finite_or_0(M), L);
      }
      ml.y = ml.y == 0.f ? 0.f : 1.f / ml.y;
    }
    s_ml[i] = ml;
  }
  __syncthreads();
  float sum = 0.f;
  for (int t0 = 0;;) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (t0 + i < tiles)
#pragma unroll
        for (int h = 0; h < PACK; ++h) {
          const float2 ml = s_ml[(t0 + i) * PACK + h];
          if (ml.y != 0.f) sum += ex2(x[i][h] - ml.x) * ml.y;
        }
    t0 += AHEAD;
    if (t0 >= tiles) break;
    load(t0);
  }
  if (live) A.weight[b * A.weight_row + s] = old + sum;
}

// ---- host

// dimensions as the kernels are built for them, and the slots of a warp's tile: 16 KB of keys and values at each
inline int padded(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
inline int tile_of(int dp) { return dp == 64 ? 32 : 16; }

struct Layout {
  int dp, unit, head_tiles, columns, pack;
  size_t part_o, part_ml, whole_ml, scores, starts, bytes;
  bool counted;  // by starts_kernel
};

inline Layout layout(const sc_kv_pages& c, int q_heads) {
  Layout l{};
  const int group = q_heads / c.kv_heads;
  l.dp = padded(c.head_dim);
  l.unit = warps_of(l.dp) * tile_of(l.dp);
  l.head_tiles = (group + HEADS - 1) / HEADS;
  for (l.pack = 1; l.pack < std::min(group, HEADS); l.pack *= 2) {}
  const int64_t slots = int64_t(c.max_pages) * c.page, units = int64_t(c.batch) * c.kv_heads * ceil_div(slots, l.unit);
  l.columns = int(std::max<int64_t>(1, std::min<int64_t>(units, std::max(1, blocks_per_sm(l.dp) * SMS / l.head_tiles))));
  const size_t parts = size_t(l.head_tiles) * l.columns * 2 * HEADS;
  auto take = [&](size_t n) {
    const size_t at = l.bytes;
    l.bytes += (n + 15) / 16 * 16;
    return at;
  };
  l.part_o = take(parts * l.dp * 4);
  l.part_ml = take(parts * 8);
  l.counted = c.batch > 2 * warps_of(l.dp) * 32;
  if (l.counted) l.starts = take((size_t(c.batch) + 1) * 4);
  if (c.weight) {
    l.whole_ml = take(size_t(c.batch) * q_heads * 8);
    l.scores = take(size_t(c.batch) * c.kv_heads * l.head_tiles * slots * l.pack * 4);
  }
  return l;
}

}  // namespace da
}  // namespace sc

using namespace sc;

extern "C" size_t sc_decode_attention_workspace(const sc_kv_pages* kv, int q_heads) {
  if (check_pages(kv) || q_heads < 1 || q_heads % kv->kv_heads || q_heads > 2048) return 0;
  return da::layout(*kv, q_heads).bytes;
}

extern "C" int sc_decode_attention(const sc_kv_pages* kv, const void* q, int64_t q_row, int64_t q_head, int q_heads,
                                   float scale, void* out, void* workspace, size_t workspace_bytes, int* err,
                                   void* stream) {
  if (int rc = check_pages(kv)) return rc;
  if (kv->batch && (!q || !out || !workspace)) return SC_ERR_ARG;
  if (q_heads < 1 || q_heads % kv->kv_heads || q_heads > 2048) return SC_ERR_SHAPE;
  if (((used(kv->batch, q_row) | used(q_heads, q_head)) & 7) ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(out)) & 15))
    return SC_ERR_ALIGN;
  const da::Layout l = da::layout(*kv, q_heads);
  if (workspace_bytes < l.bytes) return SC_ERR_WORKSPACE;
  if (kv->batch == 0) return SC_OK;
  da::Args A{};
  A.pages = pages_of(*kv);
  A.q = q, A.q_row = q_row, A.q_head = q_head;
  A.batch = kv->batch, A.q_heads = q_heads, A.kv_heads = kv->kv_heads, A.group = q_heads / kv->kv_heads;
  A.head_tiles = l.head_tiles, A.dim = kv->head_dim, A.columns = l.columns;
  A.scale_log2 = scale * 1.4426950408889634f;
  A.out = out, A.weight = kv->weight, A.weight_row = kv->weight_row;
  char* ws = static_cast<char*>(workspace);
  A.part_o = reinterpret_cast<float*>(ws + l.part_o);
  A.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
  A.slots = int64_t(kv->max_pages) * kv->page;
  A.pack = l.pack;
  if (kv->weight) {
    A.whole_ml = reinterpret_cast<float2*>(ws + l.whole_ml);
    A.scores = reinterpret_cast<float*>(ws + l.scores);
  }
  if (l.counted) A.starts = reinterpret_cast<int32_t*>(ws + l.starts);
  A.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int slot_blocks = kv->weight ? int(ceil_div(A.slots, da::JOIN_THREADS)) : 0;
  const int64_t join_blocks = int64_t(kv->batch) * (q_heads + slot_blocks);
  if (join_blocks > INT32_MAX || int64_t(kv->batch) * kv->kv_heads * ceil_div(A.slots, l.unit) > INT32_MAX) return SC_ERR_SHAPE;
  auto run = [&](auto t, auto dp, auto sub) -> int {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value, SUB = decltype(sub)::value;
    constexpr int warps = da::warps_of(DP), smem = warps * da::HEADS * DP * 4;
    const auto attend = da::attend_kernel<T, DP, SUB>;
    if (int rc = raise_smem(reinterpret_cast<const void*>(attend), smem, "decode attention smem attribute")) return rc;
    // programmatic dependent launches: blocks are placed as those of the kernel before leave
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.stream = s;
    cfg.gridDim = dim3(unsigned(l.columns), unsigned(l.head_tiles));
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = smem;
    if (l.counted) {
      da::starts_kernel<<<1, da::STARTS_THREADS, 0, s>>>(A, l.unit);
      cfg.numAttrs = 1;
    }
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, attend, A)) return cuda_failed(e, "decode attention launch");
    cfg.gridDim = dim3(unsigned(join_blocks));
    cfg.blockDim = dim3(da::JOIN_THREADS);
    cfg.dynamicSmemBytes = kv->weight ? size_t(kv->kv_heads) * l.head_tiles * l.pack * 8 : 0;
    cfg.numAttrs = 1;
    const auto join = l.pack == 1 ? da::join_kernel<T, DP, 1> : l.pack == 2 ? da::join_kernel<T, DP, 2>
                    : l.pack == 4 ? da::join_kernel<T, DP, 4> : da::join_kernel<T, DP, 8>;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, join, A, l.unit, slot_blocks))
      return cuda_failed(e, "decode attention join launch");
    if (cudaError_t e = cudaGetLastError()) return cuda_failed(e, "decode attention launch");
    return SC_OK;
  };
  auto typed = [&](auto t) -> int {
    using std::integral_constant;
    if (l.dp == 64) return run(t, integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if (l.dp == 128) return run(t, integral_constant<int, 128>{}, integral_constant<int, 1>{});
    return run(t, integral_constant<int, 256>{}, integral_constant<int, 1>{});
  };
  return kv->dtype == SC_BF16 ? typed(__nv_bfloat16{}) : typed(__half{});
}
