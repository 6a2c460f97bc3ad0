// Linear attention over prompts on the fifth-generation tensor cores (sc_linear_attention, bfloat16). In chunks of 64
// tokens, with G_i the sum of the decays of a chunk's tokens 0 .. i and S the state before the chunk:
//   out_i = scale ( e^{G_i} q_i S + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j )
//   S'    = e^{G_63} S + sum_j e^{G_63 - G_j} k_j v_j^T
// four products a chunk, with the state transposed so that value dimensions are the products' 128 rows:
//   A = Q K^T             (64 x 64)     -> P: times e^{G_i - G_j}, zero above the diagonal, rounded to bfloat16
//   I = V^T P^T           (128 x 64)    the chunk's own part of the outputs
//   X = S^T Q^T           (128 x 64)    the state's part; S^T from tensor memory as two bfloat16 terms (its rounding
//                                       and the rest), so that of the outputs only P and the result are rounded
//   D = V^T (w K)         (128 x k_dim) what the chunk adds; w_j k_j as three bfloat16 terms, exact to 2^-24
// The state stays in float32 registers: S = a S + D. A decay a near 1 enters as S + (a - 1) S, as its own rounding
// would be repeated every chunk.
//
// A block per (segment of the tokens, value head, sequence); 17 warps:
//   0-3    P from A, and the outputs            4-11   the state (a lane a value dimension, half of k_dim each)
//   12-15  loads (cp.async, three chunks in flight: any strides, zeros past a length), decays, w K
//   16     one lane issues the products
// Tensor memory: A, I, X, D and the two terms of S^T, 448 of 512 columns.
//
// One sequence's heads fill few SMs, so a long prompt is cut into segments: a first launch works out what each
// segment adds to the state (D alone), a second adds up the states before the segments, a third is the whole.
// What bounds it: a chunk's loads and stores are 64 KB at 128 dimensions (1.5 us of an SM's share of the measured
// copy), its products about 1,800 tensor cycles, and its conversions about 7,000 warp instructions.
// Every wait is bounded; one that gives up records SC_ERR_TIMEOUT and the block winds down.
#include <algorithm>
#include <type_traits>

#include "linear.cuh"
#include "tcgen05.cuh"

namespace sc {
namespace lc {

using namespace tc;

constexpr int C = 64;        // tokens of a chunk
constexpr int STAGES = 3;    // chunks loaded ahead
constexpr int RING = 4;      // chunks whose decays are held: one more, as outputs are read after a stage is free
constexpr int HALF = C * 128;  // bytes of 64 columns of a chunk's rows
constexpr int STATE_WARP = 4, LOAD_WARP = 12, MMA_WARP = 16;
constexpr int THREADS = (MMA_WARP + 1) * 32;
constexpr int SMS = 148;
constexpr float LEAST = -30.f;  // a token's decay below e^-30 is taken as e^-30: past it nothing is left in float32

// tensor memory columns
constexpr uint32_t COL_A = 0, COL_I = 64, COL_X = 128, COL_D = 192, COL_S = 320;

struct Decays {
  float g2[C], eg[C], w[C];  // G_i log2(e), e^{G_i}, e^{G_63 - G_i}
  float a, one;              // the chunk's decay as S' = a S + one S + D
};

struct Bars {
  uint64_t full[STAGES], empty[STAGES];
  uint64_t a_full, a_empty, p_full, p_empty, o_full, o_empty, kw_full, kw_empty, d_full, d_empty, s_full, s_empty, done;
  uint32_t tmem;
  int bail;
};

template <int DK>
struct Shape {
  static constexpr int K_BYTES = DK / 64 * HALF, V_BYTES = 2 * HALF;
  static constexpr int STAGE = 2 * K_BYTES + V_BYTES;
  static constexpr int KW = STAGES * STAGE, P = KW + 3 * K_BYTES, DEC = P + HALF, BARS = DEC + RING * int(sizeof(Decays));
  static constexpr int BYTES = BARS + int(sizeof(Bars)) + 1024;  // and to align the start
};

struct Args {
  sc_linear a;
  int segments, per;   // chunks of a segment
  float* parts;        // (batch, v_heads, segments, DK, 128): what a segment adds, then the state before it
  float* logs;         // (batch, v_heads, segments): the segments' decays
  int* err;
};

__device__ __forceinline__ void load16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void group_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // the loading warps

__device__ __forceinline__ uint32_t bits_of(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ float lo_f(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_f(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// the three bfloat16 terms of two float32 values
__device__ __forceinline__ void split3(float x, float y, uint32_t& t0, uint32_t& t1, uint32_t& t2) {
  t0 = bits_of(__floats2bfloat162_rn(x, y));
  x -= lo_f(t0), y -= hi_f(t0);
  t1 = bits_of(__floats2bfloat162_rn(x, y));
  t2 = bits_of(__floats2bfloat162_rn(x - lo_f(t1), y - hi_f(t1)));
}

template <int DK, bool WHOLE>
__global__ void __launch_bounds__(THREADS, 1) chunk_kernel(const __grid_constant__ Args A) {
  using L = Shape<DK>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  Decays* dec = reinterpret_cast<Decays*>(smem + L::DEC);
  Bars& B = *reinterpret_cast<Bars*>(smem + L::BARS);
  const sc_linear& a = A.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int seg = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / (a.v_heads / a.k_heads);
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.tokens) : a.tokens;
  const int c0 = seg * A.per, all = (a.tokens + C - 1) / C, c1 = min(all, c0 + A.per);
  const int n = max(0, min(c1, (len + C - 1) / C) - c0);  // this segment's chunks with tokens
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&B.full[i], 1), mbar_init(&B.empty[i], 4 + 1);
    mbar_init(&B.a_full, 1), mbar_init(&B.a_empty, 4), mbar_init(&B.p_full, 4), mbar_init(&B.p_empty, 1);
    mbar_init(&B.o_full, 1), mbar_init(&B.o_empty, 4), mbar_init(&B.kw_full, 4), mbar_init(&B.kw_empty, 1);
    mbar_init(&B.d_full, 1), mbar_init(&B.d_empty, 8), mbar_init(&B.s_full, 8), mbar_init(&B.s_empty, 1);
    mbar_init(&B.done, 1);
    B.bail = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // columns past the dimensions are never loaded: zeros
  for (int i = tid; i < L::KW / 16; i += THREADS) *reinterpret_cast<uint4*>(smem + 16 * i) = make_uint4(0, 0, 0, 0);
  fence_async();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = B.tmem;
  volatile int* bail = &B.bail;
  auto wait = [&](uint64_t* bar, int phase) -> bool {  // for the whole warp
    const bool ok = __all_sync(0xffffffffu, mbar_wait_sleep(bar, uint32_t(phase) & 1, A.err));
    if (!ok) *bail = 1;
    return ok && !*bail;
  };
  auto arrive = [&](uint64_t* bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  const uint32_t quarter = uint32_t(warp & 3) * 32, lanes = tmem + (quarter << 16);

  if (warp < STATE_WARP) {
    if constexpr (WHOLE) {
      // ---- P of the next chunk, then the outputs of this one
      const int g = lane >> 2, t = lane & 3, r0 = 16 * warp + g;
      uint8_t* p = smem + L::P;
      auto make_p = [&](int i) -> bool {
        if (!wait(&B.a_full, i)) return false;
        fence_after();
        uint32_t r[32];
        ld_frag64(lanes + COL_A, r);
        wait_ld();
        fence_before();
        arrive(&B.a_empty);
        const float* g2 = dec[i % RING].g2;
        const float ga = g2[r0], gb = g2[r0 + 8];
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 gj = *reinterpret_cast<const float2*>(g2 + 8 * j + 2 * t);
          const int col = 8 * j + 2 * t;
          auto term = [&](uint32_t x, float gi, float gk, bool in) { return in ? __uint_as_float(x) * exp2f(gi - gk) : 0.f; };
          pk[2 * j] = bits_of(__floats2bfloat162_rn(term(r[4 * j], ga, gj.x, col <= r0), term(r[4 * j + 1], ga, gj.y, col + 1 <= r0)));
          pk[2 * j + 1] = bits_of(__floats2bfloat162_rn(term(r[4 * j + 2], gb, gj.x, col <= r0 + 8),
                                                        term(r[4 * j + 3], gb, gj.y, col + 1 <= r0 + 8)));
        }
        if (!wait(&B.p_empty, i + 1)) return false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // r0 and r0 + 8 have one place in the swizzle
          *reinterpret_cast<uint32_t*>(p + r0 * 128 + ((j ^ g) << 4) + 4 * t) = pk[2 * j];
          *reinterpret_cast<uint32_t*>(p + (r0 + 8) * 128 + ((j ^ g) << 4) + 4 * t) = pk[2 * j + 1];
        }
        fence_async();
        arrive(&B.p_full);
        return true;
      };
      const int dv = int(quarter) + lane;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + (int64_t(b) * a.tokens * a.v_heads + h) * a.v_dim + dv;
      const int64_t row = int64_t(a.v_heads) * a.v_dim;
      bool ok = n == 0 || make_p(0);
      for (int i = 0; i < n && ok; ++i) {
        if (i + 1 < n && !(ok = make_p(i + 1))) break;
        if (!(ok = wait(&B.o_full, i))) break;
        fence_after();
        const int t0 = (c0 + i) * C;
        const float* eg = dec[i % RING].eg;
#pragma unroll
        for (int q = 0; q < C; q += 16) {
          uint32_t x[16], y[16];
          ld16(lanes + COL_X + q, x);
          ld16(lanes + COL_I + q, y);
          wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float o = fmaf(eg[q + e], __uint_as_float(x[e]), __uint_as_float(y[e])) * a.scale;
            if (dv < a.v_dim && t0 + q + e < a.tokens) out[(t0 + q + e) * row] = __float2bfloat16_rn(o);
          }
        }
        fence_before();
        arrive(&B.o_empty);
      }
      if (dv < a.v_dim)  // zeros past the last chunk with tokens
        for (int t1 = (c0 + n) * C; t1 < min(a.tokens, c1 * C); ++t1) out[t1 * row] = __float2bfloat16_rn(0.f);
    }
  } else if (warp < LOAD_WARP) {
    // ---- the state: value dimension `dv`, key dimensions k0 .. k0 + DK / 2 - 1
    constexpr int N = DK / 2;
    const int dv = int(quarter) + lane, k0 = (warp - STATE_WARP) / 4 * N;
    float S[N];
    const int64_t head = int64_t(b) * a.v_heads + h;
    const bool started = WHOLE && A.segments > 1;
    const float* from = started ? A.parts + (head * A.segments + seg) * DK * 128 + dv
                                : a.state_in + head * a.k_dim * a.v_dim + dv;
    const int ld = started ? 128 : a.v_dim;
#pragma unroll
    for (int k = 0; k < N; ++k)
      S[k] = WHOLE && (started || (a.state_in && dv < a.v_dim && k0 + k < a.k_dim)) ? from[int64_t(k0 + k) * ld] : 0.f;
    auto publish = [&] {  // S^T as two terms, the A operand of X
#pragma unroll
      for (int k = 0; k < N; k += 16) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = S[k + 2 * e], y = S[k + 2 * e + 1];
          hi[e] = bits_of(__floats2bfloat162_rn(x, y));
          lo[e] = bits_of(__floats2bfloat162_rn(x - lo_f(hi[e]), y - hi_f(hi[e])));
        }
        st8(lanes + COL_S + (k0 + k) / 2, hi);
        st8(lanes + COL_S + DK / 2 + (k0 + k) / 2, lo);
      }
      wait_st();
      fence_before();
      arrive(&B.s_full);
    };
    if (WHOLE && n > 0) publish();
    float log = 0.f;
    for (int i = 0; i < n; ++i) {
      if (!wait(&B.d_full, i)) break;
      fence_after();
      const float d = dec[i % RING].a, one = dec[i % RING].one;
#pragma unroll
      for (int k = 0; k < N; k += 16) {
        uint32_t r[16];
        ld16(lanes + COL_D + k0 + k, r);
        wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) S[k + e] = fmaf(d, S[k + e], fmaf(one, S[k + e], __uint_as_float(r[e])));
      }
      if (!WHOLE) log += dec[i % RING].g2[C - 1];
      fence_before();
      arrive(&B.d_empty);
      if (WHOLE && i + 1 < n) {
        if (!wait(&B.s_empty, i)) break;
        fence_after();
        publish();
      }
    }
    if (!WHOLE) {
      float* to = A.parts + (head * A.segments + seg) * DK * 128 + dv;
#pragma unroll
      for (int k = 0; k < N; ++k) to[int64_t(k0 + k) * 128] = S[k];
      if (warp == STATE_WARP && lane == 0) A.logs[head * A.segments + seg] = log * 0.69314718056f;
    } else if (seg == A.segments - 1) {
      float* to = a.state_out + head * a.k_dim * a.v_dim + dv;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (dv < a.v_dim && k0 + k < a.k_dim) to[int64_t(k0 + k) * a.v_dim] = S[k];
    }
  } else if (warp < MMA_WARP) {
    // ---- loads, decays, w K
    const int lt = tid - LOAD_WARP * 32;
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + b * a.q_row + hk * a.q_head;
    const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(a.k) + b * a.k_row + hk * a.k_head;
    const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v) + b * a.v_row + h * a.v_head;
    const float* decay = a.decay + b * a.decay_row + h * a.decay_head;
    auto issue = [&](int i) {
      const int t0 = (c0 + i) * C, m = min(C, len - t0);
      const uint32_t st = smem_u32(smem + (i % STAGES) * L::STAGE);
      auto rows = [&](uint32_t dst, const __nv_bfloat16* src, int64_t token, int pieces, auto width) {
        constexpr int W = decltype(width)::value / 8;  // 16-byte pieces of a row
#pragma unroll 4
        for (int j = lt; j < C * W; j += 128) {
          const int r = j / W, p = j % W;
          const bool in = r < m;
          if (p < pieces) load16(dst + (p >> 3) * HALF + r * 128 + (((p & 7) ^ (r & 7)) << 4), in ? src + (t0 + r) * token + 8 * p : src, in);
        }
      };
      rows(st + L::K_BYTES, k, a.k_token, a.k_dim / 8, std::integral_constant<int, DK>{});
      if (WHOLE) rows(st, q, a.q_token, a.k_dim / 8, std::integral_constant<int, DK>{});
      rows(st + 2 * L::K_BYTES, v, a.v_token, a.v_dim / 8, std::integral_constant<int, 128>{});
    };
    auto commit_group = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    auto decay_of = [&](int i, int e) -> float {
      const int t = (c0 + i) * C + 2 * lane + e;
      return i < n && t < len ? fmaxf(decay[int64_t(t) * a.decay_token], LEAST) : 0.f;
    };
    float d0 = 0.f, d1 = 0.f;
    if (warp == LOAD_WARP) d0 = decay_of(0, 0), d1 = decay_of(0, 1);
    for (int i = 0; i < STAGES - 1; ++i) {
      if (i < n) issue(i);
      commit_group();
    }
    for (int i = 0; i < n; ++i) {
      Decays& D = dec[i % RING];
      if (warp == LOAD_WARP) {  // tokens 2 lane and 2 lane + 1: sums from the front, and from the back
        const float g0 = d0, g1 = d1, pair = g0 + g1;
        d0 = decay_of(i + 1, 0), d1 = decay_of(i + 1, 1);
        float up = pair, down = pair;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float x = __shfl_up_sync(0xffffffffu, up, o), y = __shfl_down_sync(0xffffffffu, down, o);
          if (lane >= o) up += x;
          if (lane + o < 32) down += y;
        }
        float before = __shfl_up_sync(0xffffffffu, up, 1), after = __shfl_down_sync(0xffffffffu, down, 1);
        if (lane == 0) before = 0.f;
        if (lane == 31) after = 0.f;
        constexpr float LOG2E = 1.4426950408889634f;
        const float e0 = (before + g0) * LOG2E, e1 = up * LOG2E;
        *reinterpret_cast<float2*>(&D.g2[2 * lane]) = make_float2(e0, e1);
        *reinterpret_cast<float2*>(&D.eg[2 * lane]) = make_float2(exp2f(e0), exp2f(e1));
        *reinterpret_cast<float2*>(&D.w[2 * lane]) = make_float2(exp2f((after + g1) * LOG2E), exp2f(after * LOG2E));
        if (lane == 31) {
          const bool near = up > -0.69314718f;
          D.a = near ? expm1f(up) : expf(up), D.one = near ? 1.f : 0.f;
        }
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      fence_async();
      group_sync();
      const int st = i % STAGES;
      if (lt == 0) mbar_arrive(&B.full[st]);
      if (!wait(&B.kw_empty, i + 1)) break;
      const uint8_t* kr = smem + st * L::STAGE + L::K_BYTES;
      uint8_t* kw = smem + L::KW;
#pragma unroll 2
      for (int j = lt; j < C * DK / 8; j += 128) {  // 16 bytes of K at a time, the terms to the same places
        const int at = j * 16, r = (at % HALF) / 128;
        const uint4 x = *reinterpret_cast<const uint4*>(kr + at);
        const float w = D.w[r];
        uint4 t0, t1, t2;
        split3(lo_f(x.x) * w, hi_f(x.x) * w, t0.x, t1.x, t2.x);
        split3(lo_f(x.y) * w, hi_f(x.y) * w, t0.y, t1.y, t2.y);
        split3(lo_f(x.z) * w, hi_f(x.z) * w, t0.z, t1.z, t2.z);
        split3(lo_f(x.w) * w, hi_f(x.w) * w, t0.w, t1.w, t2.w);
        *reinterpret_cast<uint4*>(kw + at) = t0;
        *reinterpret_cast<uint4*>(kw + L::K_BYTES + at) = t1;
        *reinterpret_cast<uint4*>(kw + 2 * L::K_BYTES + at) = t2;
      }
      fence_async();
      arrive(&B.kw_full);
      arrive(&B.empty[st]);  // K has been read
      // the next chunk's loads, into the stage of the chunk before this one
      const int ahead = i + STAGES - 1;
      if (ahead < n) {
        if (ahead >= STAGES && !wait(&B.empty[ahead % STAGES], ahead / STAGES - 1)) break;
        issue(ahead);
      }
      commit_group();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---- the products
    const bool leader = elect_one();
    auto k_major = [&](const uint8_t* p, int s) { return desc_k(p + (s / 4) * HALF) + 2 * (s % 4); };
    auto a_product = [&](int i) {
      const uint8_t* st = smem + (i % STAGES) * L::STAGE;
      if (leader) {
#pragma unroll
        for (int s = 0; s < DK / 16; ++s)
          mma_ss(tmem + COL_A, k_major(st, s), k_major(st + L::K_BYTES, s), idesc_bf16(64, 64, false, false), s > 0);
        commit(&B.a_full);
      }
      __syncwarp();
    };
    bool ok = true;
    if (WHOLE && n > 0 && (ok = wait(&B.full[0], 0))) {
      fence_after();
      a_product(0);
    }
    for (int i = 0; i < n && ok; ++i) {
      const int st = i % STAGES;
      const uint8_t* stage = smem + st * L::STAGE;
      const uint64_t vt = desc_mn(stage + 2 * L::K_BYTES, HALF);
      if (!(ok = wait(&B.full[st], i / STAGES))) break;
      if (!(ok = wait(&B.kw_full, i))) break;
      if (!(ok = wait(&B.d_empty, i + 1))) break;
      fence_after();
      if (leader) {
#pragma unroll
        for (int term = 2; term >= 0; --term)  // the small ones first
#pragma unroll
          for (int s = 0; s < C / 16; ++s)
            mma_ss(tmem + COL_D, vt + 128 * s, desc_mn(smem + L::KW + term * L::K_BYTES, HALF) + 128 * s,
                   idesc_bf16(128, DK, true, true), term < 2 || s > 0);
        commit(&B.d_full);
        commit(&B.kw_empty);
        if (!WHOLE) commit(&B.empty[st]);
      }
      __syncwarp();
      if constexpr (WHOLE) {
        if (!(ok = wait(&B.s_full, i))) break;
        if (!(ok = wait(&B.o_empty, i + 1))) break;
        fence_after();
        if (leader) {
#pragma unroll
          for (int term = 1; term >= 0; --term)
#pragma unroll
            for (int s = 0; s < DK / 16; ++s)
              mma_ts(tmem + COL_X, tmem + COL_S + term * (DK / 2) + 8 * s, k_major(stage, s), idesc_bf16(128, 64, false, false),
                     term < 1 || s > 0);
          commit(&B.s_empty);
        }
        __syncwarp();
        if (i + 1 < n) {
          if (!(ok = wait(&B.full[(i + 1) % STAGES], (i + 1) / STAGES))) break;
          if (!(ok = wait(&B.a_empty, i))) break;
          fence_after();
          a_product(i + 1);
        }
        if (!(ok = wait(&B.p_full, i))) break;
        fence_after();
        if (leader) {
#pragma unroll
          for (int s = 0; s < C / 16; ++s)
            mma_ss(tmem + COL_I, vt + 128 * s, desc_k(smem + L::P) + 2 * s, idesc_bf16(128, 64, true, false), s > 0);
          commit(&B.o_full);
          commit(&B.p_empty);
          commit(&B.empty[st]);
        }
        __syncwarp();
      }
    }
    if (leader) {
      commit(&B.done);  // every product issued has finished
      mbar_wait(&B.done, 0, nullptr, 20000000LL);
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// the states before the segments, in place of what the segments add: a thread a value
template <int DK>
__global__ void __launch_bounds__(256) scan_kernel(const Args A) {
  const sc_linear& a = A.a;
  const int64_t head = blockIdx.x;
  const int e = blockIdx.y * 256 + threadIdx.x, k = e / 128, dv = e % 128;
  float* part = A.parts + head * A.segments * DK * 128 + e;
  float S = a.state_in && k < a.k_dim && dv < a.v_dim ? a.state_in[(head * a.k_dim + k) * a.v_dim + dv] : 0.f;
#pragma unroll 4
  for (int s = 0; s + 1 < A.segments; ++s) {
    const float log = A.logs[head * A.segments + s], add = part[int64_t(s) * DK * 128];
    part[int64_t(s) * DK * 128] = S;
    S = log > -0.69314718f ? fmaf(expm1f(log), S, S + add) : fmaf(expf(log), S, add);
  }
  part[int64_t(A.segments - 1) * DK * 128] = S;
}

// The segments that cost least: waves of blocks times a segment's chunks, those of the first launch (about two fifths
// of the whole's work each) added, and 10 chunks' time for the two more launches.
inline int segments_of(const sc_linear& a) {
  const int64_t heads = int64_t(a.batch) * a.v_heads;
  const int chunks = int(ceil_div(a.tokens, C));
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= std::min(chunks / 4, SMS) || s == 1; ++s) {
    const double per = double(ceil_div(chunks, s)), waves = double(ceil_div(heads * s, SMS));
    const double cost = waves * per + (s > 1 ? 0.4 * double(ceil_div(heads * (s - 1), SMS)) * per + 10 : 0);
    if (cost < least) least = cost, best = s;
  }
  return best;
}

inline size_t parts_bytes(const sc_linear& a, int segments) {
  const int dk = a.k_dim <= 64 ? 64 : 128;
  return segments > 1 ? size_t(a.batch) * a.v_heads * segments * (size_t(dk) * 128 + 4) * 4 : 0;
}

size_t workspace(const sc_linear& a) { return parts_bytes(a, segments_of(a)) + 16; }

template <int DK>
int run(const Args& A, cudaStream_t s) {
  const sc_linear& a = A.a;
  const dim3 grid(unsigned(A.segments), unsigned(a.v_heads), unsigned(a.batch));
  constexpr int smem = Shape<DK>::BYTES;
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  if (int rc = raise_smem(reinterpret_cast<const void*>(chunk_kernel<DK, true>), smem, "linear attention smem attribute"))
    return rc;
  if (A.segments > 1) {
    if (int rc = raise_smem(reinterpret_cast<const void*>(chunk_kernel<DK, false>), smem, "linear attention smem attribute"))
      return rc;
    chunk_kernel<DK, false><<<dim3(grid.x - 1, grid.y, grid.z), THREADS, smem, s>>>(A);
    scan_kernel<DK><<<dim3(unsigned(a.batch) * unsigned(a.v_heads), DK * 128 / 256), 256, 0, s>>>(A);
  }
  chunk_kernel<DK, true><<<grid, THREADS, smem, s>>>(A);
  if (cudaError_t e = cudaGetLastError()) return cuda_failed(e, "linear attention launch");
  return SC_OK;
}

int launch(const sc_linear& a, void* ws, int* err, cudaStream_t s) {
  Args A{};
  A.a = a;
  A.segments = segments_of(a);
  A.per = int(ceil_div(ceil_div(a.tokens, C), A.segments));
  const int dk = a.k_dim <= 64 ? 64 : 128;
  A.parts = static_cast<float*>(ws);
  A.logs = A.parts + size_t(a.batch) * a.v_heads * A.segments * dk * 128;
  A.err = err;
  return dk == 64 ? run<64>(A, s) : run<128>(A, s);
}

}  // namespace lc
}  // namespace sc
