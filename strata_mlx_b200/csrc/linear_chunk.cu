// Linear attention over prompts on the fifth-generation tensor cores (sc_linear_attention, bfloat16). In chunks of 64
// tokens, with G_i the sum of the decays of a chunk's tokens 0 .. i and S the state before the chunk:
//   out_i = scale ( e^{G_i} q_i S + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j )
//   S'    = e^{G_63} S + sum_j e^{G_63 - G_j} k_j v_j^T
// four products a chunk, with the state transposed so that value dimensions are the products' 128 rows:
//   A = Q K^T             (64 x 64)     -> P: times e^{G_i - G_j}, zero above the diagonal
//   I = V^T P^T           (128 x 64)    the chunk's own part of the outputs; P as two bfloat16 terms, its rounding and
//                                       what that left (one term alone made the outputs' error 1.4 times their rounding)
//   X = S^T Q^T           (128 x 64)    the state's part; S^T from tensor memory as two terms too, so that of the
//                                       outputs only the result is rounded
//   D = V^T (w K)         (128 x k_dim) what the chunk adds; w_j k_j as three bfloat16 terms, exact to 2^-24
// The state stays in float32 registers: S = a S + D. A decay a near 1 (between a half and two) enters as S + (a - 1) S,
// as its own rounding would be repeated every chunk.
//
// A block per (segment of the tokens, value head, sequence); 24 warps in six groups, each with its share of registers:
//   0-3    P from A                             4-7    the outputs, stored by TMA through a tile in shared memory
//   8-15   the state (a lane a value dimension, half of k_dim each)
//   16-19  w K, in halves of 32 tokens so that D's products run behind it; zeros over the values past a length
//   20     one lane issues A, X and I           21  the chunks' decays; loads of values
//   22     loads of queries and keys            23  one lane issues D
// Tensor memory: A, I, two of X, D and the two terms of S^T, all 512 columns.
//
// One sequence's heads fill few SMs, so a long prompt is cut into segments: a first launch works out what each
// segment adds to the state, a second adds up the states before the segments, a third is the whole. The first takes a
// segment's chunks from the last to the first, the weights w running on from chunk to chunk, so that D of eight chunks
// adds up in tensor memory and no state is carried between them.
// What bounds it at 128 dimensions, a chunk: 64 KB of loads and stores (1.5 us of an SM's share of the measured copy),
// 1,792 tensor cycles (A, of 64 rows, runs at half rate), 9,800 warp instructions (2,450 cycles of issue), and the chain
// state -> its terms -> X -> state, which sets the pace: 3,500 cycles where a block is alone, 3,900 with all SMs at work.
// A loop's code counts twice: 24 warps in eight roles share the instruction cache, and what does not fit is fetched
// again every chunk (kernel of 116 KB: 282 us for 32768 tokens of 16 heads, 70 KB: 195, 61 KB: 184). So loops are rolled, an
// operation stands in one place, and both halves of P run through the same code.
// Every wait is bounded; one that gives up records SC_ERR_TIMEOUT and the block winds down.
#include <algorithm>
#include <type_traits>

#include "linear.cuh"
#include "tensor_map.cuh"
#include "tcgen05.cuh"

namespace sc {
namespace lc {

using namespace tc;

constexpr int C = 64;        // tokens of a chunk
// chunks of queries, keys and values held: scores are made a chunk ahead and a chunk's queries are needed until its
// last products, keys until w K is made, values for the chunk's own products only
constexpr int QS = 3, KS = 3, VS = 2;
constexpr int RING = 4;      // chunks whose decays are held
constexpr int AHEAD = 8;     // and those whose decays are fetched ahead
constexpr int HALF = C * 128;  // bytes of 64 columns of a chunk's rows
constexpr int THREADS = 24 * 32;
constexpr int OUT_WARP = 4, STATE_WARP = 8, KW_WARP = 16, MMA_WARP = 20, DECAY_WARP = 21, LOAD_WARP = 22, SUM_WARP = 23;
// registers a thread: 80 at launch; the groups' shares add up to as many
constexpr int P_REGS = 64, OUT_REGS = 56, STATE_REGS = 120, KW_REGS = 72, CONTROL_REGS = 48;
static_assert(P_REGS + OUT_REGS + 2 * STATE_REGS + KW_REGS + CONTROL_REGS == 6 * 80, "a block's registers");
// the first launch's: 12 warps make w K, 8 add up D, 3 control
constexpr int ADD_SUM_WARP = 12, ADD_KW_WARPS = 6, ADD_STAGES = 4, ADD_RUN = 8;  // chunks whose D adds up in tensor memory
constexpr int ADD_RING = 6, ADD_AHEAD = 3;  // chunks whose decays, then weights are held, and of them those fetched ahead
constexpr int SUM_REGS = 96;
static_assert(3 * 80 + 2 * SUM_REGS + CONTROL_REGS <= 6 * 80, "a block's registers");
constexpr int SMS = 148;
constexpr float LEAST = -104.f;  // a token whose decay is below this is a reset: e^-104 is zero in float32

// tensor memory columns
constexpr uint32_t COL_A = 0, COL_I = 64, COL_D = 192, COL_S = 320;
__device__ __forceinline__ uint32_t col_x(int i) { return i & 1 ? 448 : 128; }  // of chunk i: two, taken in turn

// Resets count as 0 in the sums G, so that the other tokens' differences stay exact and finite; what a reset parts is set
// to zero beside them: P by from[i], the scale e^{G_i} behind the first, the weights before the last, the chunk's a.
struct Decays {
  float g2[C], eg[C], w[C];  // G_i log2(e), scale e^{G_i}, e^{G_63 - G_i}
  float a, one;              // the chunk's decay as S' = a S + one S + D
  uint32_t resets, unused;   // whether the chunk has any
  uint8_t from[C];           // where it has: the first token that token i sees, its own or the last reset's at or before i
};

struct Bars {
  uint64_t qk_full[2][KS], qk_empty[2][KS], v_full[VS], v_empty[VS], dec_full[RING], dec_empty[RING];
  uint64_t a_full, a_empty, p_full, p_empty, o_full, o_empty, kw_full[2], kw_empty[2], d_full, d_empty, s_full, s_empty,
      ends, outs, done;
  uint32_t tmem;
  int bail;
  int odd[4];  // whether a state at the segment's end is not finite, for each quarter of the value dimensions
};

struct AddBars {
  uint64_t full[ADD_STAGES], empty[ADD_STAGES], dec_full[ADD_RING], dec_empty[ADD_RING], kw_full[2], kw_empty[2], d_full[2],
      d_empty[2], done;
  uint32_t tmem;
  int bail;
};

// chunk i's place in a ring, and the phase of its barriers
template <int N> __device__ __forceinline__ uint32_t slot(int i) { return uint32_t(i) % N; }
template <int N> __device__ __forceinline__ int phase(int i) { return int(uint32_t(i) / N); }

template <int DK>
struct Shape {
  static constexpr int K_BYTES = DK / 64 * HALF, V_BYTES = 2 * HALF;
  static constexpr int Q = 0, K = Q + QS * K_BYTES, V = K + KS * K_BYTES, KW = V + VS * V_BYTES, P = KW + 3 * K_BYTES;
  static constexpr int OUT = P + 2 * HALF, DEC = OUT + V_BYTES, RAW = DEC + RING * int(sizeof(Decays));
  static constexpr int BARS = RAW + AHEAD * C * 4;
  static constexpr int BYTES = BARS + int(sizeof(Bars)) + 1024;  // and to align the start
};
template <int DK>
struct AddShape {
  static constexpr int K_BYTES = DK / 64 * HALF, V_BYTES = 2 * HALF, STAGE = K_BYTES + V_BYTES;
  static constexpr int KW = ADD_STAGES * STAGE, DEC = KW + 2 * 3 * K_BYTES, BARS = DEC + ADD_RING * C * 4;
  static constexpr int BYTES = BARS + int(sizeof(AddBars)) + 1024;
};

struct Args {
  sc_linear a;
  int segments, per;   // chunks of a segment
  float* parts;        // (batch, v_heads, segments, DK, 128): what a segment adds, then the state before it
  float* logs;         // (batch, v_heads, segments): the segments' decays
  int* err;
};

struct Maps {  // (dim, heads, tokens, batch), boxes of 64 x 1 x 64 x 1, 128-byte swizzle
  CUtensorMap q, k, v, out;
};

__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int h, int t, int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(h), "r"(t), "r"(b), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, const void* src, int x, int h, int t, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(h), "r"(t), "r"(b), "r"(smem_u32(src))
               : "memory");
}
// four 8 x 8 fragments, transposed, to the rows whose addresses the lanes give
__device__ __forceinline__ void store_transposed(uint32_t at, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r0), "r"(r1), "r"(r2),
               "r"(r3)
               : "memory");
}
// the output warps; whether all of them go on: one that gave up its wait would leave the others at the barrier
__device__ __forceinline__ void out_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool out_all(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(uint32_t(ok))
      : "memory");
  return all != 0;
}

__device__ __forceinline__ uint32_t bits_of(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ float lo_f(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_f(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// 2^x to 2^-22 of it, zero below 2^-126: P is rounded to eight bits, and a token's weight carries no further
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// e^x - 1 for x in [-ln 2, ln 2], by its series to x^10 / 10!: within 2^-28 of it
__device__ __forceinline__ float expm1_near(float x) {
  float y = 1.f / 3628800.f;
  y = fmaf(y, x, 1.f / 362880.f);
  y = fmaf(y, x, 1.f / 40320.f);
  y = fmaf(y, x, 1.f / 5040.f);
  y = fmaf(y, x, 1.f / 720.f);
  y = fmaf(y, x, 1.f / 120.f);
  y = fmaf(y, x, 1.f / 24.f);
  y = fmaf(y, x, 1.f / 6.f);
  y = fmaf(y, x, 0.5f);
  return fmaf(y * x, x, x);
}

__device__ __forceinline__ float2 unpacked(uint32_t v) { return make_float2(lo_f(v), hi_f(v)); }
__device__ __forceinline__ uint32_t rounded(float2 v) { return bits_of(__floats2bfloat162_rn(v.x, v.y)); }
// two values less their bfloat16 roundings, exactly
__device__ __forceinline__ float2 rest(float2 v, uint32_t r) { return __ffma2_rn(unpacked(r), make_float2(-1.f, -1.f), v); }

// the three bfloat16 terms of two float32 values
__device__ __forceinline__ void split3(float2 v, uint32_t& t0, uint32_t& t1, uint32_t& t2) {
  t0 = rounded(v);
  v = rest(v, t0);
  t1 = rounded(v);
  t2 = rounded(rest(v, t1));
}

// tries of several barriers at once, so that their latencies overlap
__device__ __forceinline__ bool try_wait2(uint64_t* x, uint32_t px, uint64_t* y, uint32_t py) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
      "and.pred p, p, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(x)), "r"(px & 1), "r"(smem_u32(y)), "r"(py & 1)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool try_wait3(uint64_t* x, uint32_t px, uint64_t* y, uint32_t py, uint64_t* z, uint32_t pz) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q, r;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n\t"
      "and.pred p, p, q;\n\t"
      "and.pred p, p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(x)), "r"(px & 1), "r"(smem_u32(y)), "r"(py & 1), "r"(smem_u32(z)), "r"(pz & 1)
      : "memory");
  return ok != 0;
}

// Waits, for a whole warp (all of its lanes go on, or none) and for one thread. Small in code, as there are many: the
// warps' instructions have to fit the cache.
struct Waits {
  volatile int* bail;  // the block's; whoever finds it set stops waiting, and a thread records the error at the end
  __device__ __forceinline__ bool over(uint32_t start) const { return *bail || uint32_t(clock()) - start > 2000000000u; }
  __device__ __forceinline__ bool stop() const {
    *bail = 1;
    return false;
  }
  __device__ __forceinline__ bool operator()(uint64_t* x, int px) const {
    const uint32_t start = uint32_t(clock());
    while (!__all_sync(0xffffffffu, mbar_try_wait(x, uint32_t(px) & 1)))
      if (__any_sync(0xffffffffu, over(start))) return stop();
    return true;
  }
  // several barriers side by side
  __device__ __forceinline__ bool operator()(uint64_t* x, int px, uint64_t* y, int py) const {
    const uint32_t start = uint32_t(clock());
    while (!__all_sync(0xffffffffu, try_wait2(x, px, y, py)))
      if (__any_sync(0xffffffffu, over(start))) return stop();
    return true;
  }
  __device__ __forceinline__ bool operator()(uint64_t* x, int px, uint64_t* y, int py, uint64_t* z, int pz) const {
    const uint32_t start = uint32_t(clock());
    while (!__all_sync(0xffffffffu, try_wait3(x, px, y, py, z, pz)))
      if (__any_sync(0xffffffffu, over(start))) return stop();
    return true;
  }
  __device__ __forceinline__ bool alone(uint64_t* bar, int phase) const {
    const uint32_t start = uint32_t(clock());
    while (!mbar_try_wait(bar, uint32_t(phase) & 1))
      if (over(start)) return stop();
    return true;
  }
};
__device__ __forceinline__ void arrive(uint64_t* bar) {  // a warp's
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

__device__ __forceinline__ void tmem_alloc(uint32_t* at) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(at)), "r"(512) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(512));
}

// 16 bytes of K times w as three terms of 16 bytes, at one place of three tiles; zeros where `in` is not set
__device__ __forceinline__ void split_piece(const uint8_t* k, float w, bool in, uint8_t* to, int term) {
  uint4 x = *reinterpret_cast<const uint4*>(k);
  if (!in) x = make_uint4(0, 0, 0, 0);
  const float2 w2 = make_float2(w, w);
  uint4 t0, t1, t2;
  split3(__fmul2_rn(unpacked(x.x), w2), t0.x, t1.x, t2.x);
  split3(__fmul2_rn(unpacked(x.y), w2), t0.y, t1.y, t2.y);
  split3(__fmul2_rn(unpacked(x.z), w2), t0.z, t1.z, t2.z);
  split3(__fmul2_rn(unpacked(x.w), w2), t0.w, t1.w, t2.w);
  *reinterpret_cast<uint4*>(to) = t0;
  *reinterpret_cast<uint4*>(to + term) = t1;
  *reinterpret_cast<uint4*>(to + 2 * term) = t2;
}

// values past the length meet zeros of P and w K, which a NaN would spoil: zeros in their place, by `step` threads
__device__ __forceinline__ void clear_values(uint8_t* v, int m, int thread, int step) {
#pragma unroll 1
  for (int j = thread; j < 2 * HALF / 16; j += step)
    if ((j * 16 % HALF) / 128 >= m) *reinterpret_cast<uint4*>(v + 16 * j) = make_uint4(0, 0, 0, 0);
}

// the second half of the values is not loaded where there are 64 or fewer: zeros
__device__ __forceinline__ void clear_halves(uint8_t* v, int n, int apart) {
#pragma unroll 1
  for (int i = threadIdx.x; i < n * HALF / 16; i += THREADS)
    *reinterpret_cast<uint4*>(v + i / (HALF / 16) * apart + HALF + 16 * (i % (HALF / 16))) = make_uint4(0, 0, 0, 0);
  fence_async();
}

// D += V^T (w K): the half `hf` of the tokens, the small terms first. Here and below two to four products an iteration:
// their issue keeps ahead of the tensor cores, and the code stays small.
template <int DK>
__device__ __forceinline__ void add_products(uint32_t d, uint64_t v, uint64_t kw, int hf, bool first) {
  v += 256 * hf, kw += 256 * hf + uint32_t(2 * (DK / 64) * (HALF >> 4));
#pragma unroll 1
  for (int term = 2; term >= 0; --term, kw -= uint32_t(DK / 64 * (HALF >> 4))) {
    mma_ss(d, v, kw, idesc_bf16(128, DK, true, true), !first || term < 2);
    mma_ss(d, v + 128, kw + 128, idesc_bf16(128, DK, true, true), true);
  }
}

// A chunk's decays on their way to shared memory, a lane tokens 2 lane and 2 lane + 1 from t0 on; zeros past the length.
// Several chunks' are under way: with one, its trip to memory (2,000 cycles under load) was what a chunk took.
__device__ __forceinline__ void fetch_decays(float* place, const float* decay, int64_t token, int t0, int len) {
  const int lane = threadIdx.x & 31, t = t0 + 2 * lane;
  const uint32_t to = smem_u32(place + 2 * lane);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const bool in = t + e < len;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 4 * e), "l"(decay + (in ? (t + e) * token : 0)),
                 "r"(in ? 4 : 0)
                 : "memory");
  }
}
__device__ __forceinline__ void close_fetch() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// those of the oldest chunk under way, `Behind` chunks being behind it
template <int Behind>
__device__ __forceinline__ float2 fetched(const float* place) {
  asm volatile("cp.async.wait_group %0;" ::"n"(Behind) : "memory");
  return *reinterpret_cast<const float2*>(place + 2 * (threadIdx.x & 31));
}
// Takes the resets out of a lane's two decays; which lanes had one at their first token, and at their second. (A NaN is
// none: it goes into the sums.)
__device__ __forceinline__ uint2 take_resets(float2& g) {
  const bool x = g.x < LEAST, y = g.y < LEAST;
  if (x) g.x = 0.f;
  if (y) g.y = 0.f;
  return make_uint2(__ballot_sync(0xffffffffu, x), __ballot_sync(0xffffffffu, y));
}

// A value that is not finite meets P's zeros (0 times it is NaN) and so reaches the tokens before it in its chunk. It stays
// in the state, whatever follows; so a segment whose state at its end is finite had none, and the chunks need not look (in
// the output warps a look through a chunk's values took 2.3 of 54 us, in others more). In another segment the outputs are
// mended behind its last chunk: the recurrence from the state before the segment up to the last token whose value is the
// first that is not finite of its dimension, a lane a dimension, the state in two places of shared memory that the products
// have done with. What is not finite among the outputs and is in the recurrence is replaced. Measured: 3 us a token
// (one prompt of 32768 tokens, 16 heads, with a NaN near its end 11.8 ms, without 0.22).
template <int DK>
__device__ __forceinline__ void mend_outputs(const Args& A, uint8_t* place0, uint8_t* place1, int dv, int t0, int t1) {
  const sc_linear& a = A.a;
  const int seg = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / (a.v_heads / a.k_heads);
  const bool live = dv < a.v_dim;
  const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v) + b * a.v_row + h * a.v_head + (live ? dv : 0);
  int odd = INT32_MAX;  // the dimension's first token with such a value
#pragma unroll 8
  for (int t = t0; t < t1; ++t)
    if (!isfinite(__bfloat162float(v[t * a.v_token]))) odd = min(odd, t);
  if (!live) odd = INT32_MAX;
  const int first = __reduce_min_sync(0xffffffffu, odd) / C * C;
  const int last = __reduce_max_sync(0xffffffffu, odd == INT32_MAX ? t0 : odd);
  if (last == t0) return;
  constexpr int FIRST = QS * DK / 64 * HALF / 512;  // rows of 128 values in place0
  static_assert((DK - FIRST) * 512 <= 2 * HALF && FIRST % 8 == 0, "the state's places");
  auto S = [&](int k) -> float& { return reinterpret_cast<float*>(k < FIRST ? place0 + 512 * k : place1 + 512 * (k - FIRST))[dv]; };
  const int64_t head = int64_t(b) * a.v_heads + h;
  if (A.segments > 1) pdl_wait();
#pragma unroll 1
  for (int k = 0; k < a.k_dim; ++k) {
    float s = 0.f;
    if (A.segments > 1) s = A.parts[((head * A.segments + seg) * DK + k) * 128 + dv];
    else if (a.state_in && live) s = a.state_in[(head * a.k_dim + k) * a.v_dim + dv];
    S(k) = s;
  }
#pragma unroll 1
  for (int t = t0; t < last; ++t) {
    const __nv_bfloat16* kt = static_cast<const __nv_bfloat16*>(a.k) + b * a.k_row + hk * a.k_head + t * a.k_token;
    const float x = live ? __bfloat162float(v[t * a.v_token]) : 0.f;
    const float g = a.decay[b * a.decay_row + h * a.decay_head + t * a.decay_token];
    const bool near = fabsf(g) < 0.69314718f;
    const float d = near ? expm1_near(g) : expf(g), one = near ? 1.f : 0.f;
#pragma unroll 1
    for (int k = 0; k < a.k_dim; k += 8) {  // loads before stores: they would wait for one another
      const uint4 k8 = *reinterpret_cast<const uint4*>(kt + k);
      const uint32_t w[4] = {k8.x, k8.y, k8.z, k8.w};
      float* at = &S(k);
      float r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = at[128 * e];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = fmaf(d, r[e], fmaf(one, r[e], (e & 1 ? hi_f(w[e / 2]) : lo_f(w[e / 2])) * x));
#pragma unroll
      for (int e = 0; e < 8; ++e) at[128 * e] = r[e];
    }
    if (t < first) continue;
    const __nv_bfloat16* qt = static_cast<const __nv_bfloat16*>(a.q) + b * a.q_row + hk * a.q_head + t * a.q_token;
    float o = 0.f;
#pragma unroll 1
    for (int k = 0; k < a.k_dim; k += 2) {
      const uint32_t q2 = *reinterpret_cast<const uint32_t*>(qt + k);
      o = fmaf(lo_f(q2), S(k), fmaf(hi_f(q2), S(k + 1), o));
    }
    o *= a.scale;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + ((int64_t(b) * a.tokens + t) * a.v_heads + h) * a.v_dim + dv;
    if (live && isfinite(o) && !isfinite(__bfloat162float(*out))) *out = __float2bfloat16_rn(o);
  }
}

// What a segment adds to the state, and its decay.
template <int DK>
__global__ void __launch_bounds__(THREADS, 1) add_kernel(const __grid_constant__ Args A, const __grid_constant__ Maps maps) {
  using L = AddShape<DK>;
  extern __shared__ uint8_t raw[];
  // 1024-byte aligned, by an offset: through an integer the pointer would no longer be known to be shared memory's
  uint8_t* smem = raw + (0u - smem_u32(raw) & 1023u);
  float* dec = reinterpret_cast<float*>(smem + L::DEC);  // (ADD_RING, C) decays, then weights
  AddBars& B = *reinterpret_cast<AddBars*>(smem + L::BARS);
  const sc_linear& a = A.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int seg = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / (a.v_heads / a.k_heads);
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.tokens) : a.tokens;
  const int c0 = seg * A.per, n = max(0, min(c0 + A.per, (len + C - 1) / C) - c0);
  pdl_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < ADD_STAGES; ++i) mbar_init(&B.full[i], 1), mbar_init(&B.empty[i], ADD_KW_WARPS + 1);
    for (int i = 0; i < ADD_RING; ++i) mbar_init(&B.dec_full[i], 1), mbar_init(&B.dec_empty[i], ADD_KW_WARPS);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B.kw_full[i], ADD_KW_WARPS), mbar_init(&B.kw_empty[i], 1);
      mbar_init(&B.d_full[i], 1), mbar_init(&B.d_empty[i], 8);
    }
    mbar_init(&B.done, 1);
    B.bail = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) tmem_alloc(&B.tmem);
  if (a.v_dim <= 64) clear_halves(smem + L::K_BYTES, ADD_STAGES, L::STAGE);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = B.tmem;
  const Waits wait{&B.bail};
  auto chunk = [&](int i) { return c0 + n - 1 - i; };  // the last first
  if (warp < ADD_SUM_WARP) {
    // ---- w K, two groups of warps taking the chunks in turn: one's waits pass while the other computes
    constexpr int GROUP = ADD_KW_WARPS * 32;
    const int gt = tid % GROUP;
#pragma unroll 1
    for (int i = tid / GROUP; i < n; i += 2) {
      const int st = slot<ADD_STAGES>(i), m = len - chunk(i) * C;
      if (!wait(&B.dec_full[slot<ADD_RING>(i)], phase<ADD_RING>(i), &B.full[st], phase<ADD_STAGES>(i), &B.kw_empty[i & 1], i / 2 + 1)) break;
      const float* w = dec + slot<ADD_RING>(i) * C;
      uint8_t* kw = smem + L::KW + (i & 1) * 3 * L::K_BYTES;
#pragma unroll 2
      for (int j = gt; j < C * DK / 8; j += GROUP) {
        const int r = (j * 16 % HALF) / 128;
        split_piece(smem + st * L::STAGE + 16 * j, w[r], r < m, kw + 16 * j, L::K_BYTES);
      }
      if (m < C) clear_values(smem + st * L::STAGE + L::K_BYTES, m, gt, GROUP);
      fence_async();
      arrive(&B.kw_full[i & 1]);
      arrive(&B.empty[st]);
      arrive(&B.dec_empty[slot<ADD_RING>(i)]);
    }
  } else if (warp < MMA_WARP) {
    // ---- the sums of ADD_RUN chunks into one
    more_registers<SUM_REGS>();
    constexpr int N = DK / 2;
    const uint32_t quarter = uint32_t(warp & 3) * 32, lanes = tmem + (quarter << 16);
    const int dv = int(quarter) + lane, k0 = (warp - ADD_SUM_WARP) / 4 * N;
    float S[N];
#pragma unroll
    for (int k = 0; k < N; ++k) S[k] = 0.f;
#pragma unroll 1
    for (int r = 0; r * ADD_RUN < n; ++r) {
      if (!wait(&B.d_full[r & 1], r / 2)) break;
      fence_after();
#pragma unroll
      for (int k = 0; k < N; k += 16) {
        uint32_t x[16];
        ld16(lanes + (r & 1) * 128 + k0 + k, x);
        wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) S[k + e] += __uint_as_float(x[e]);
      }
      fence_before();
      arrive(&B.d_empty[r & 1]);
    }
    float* to = A.parts + ((int64_t(b) * a.v_heads + h) * A.segments + seg) * DK * 128 + dv;
#pragma unroll
    for (int k = 0; k < N; ++k) to[int64_t(k0 + k) * 128] = S[k];
  } else {
    fewer_registers<CONTROL_REGS>();
    if (warp == DECAY_WARP) {
      const float* decay = a.decay + b * a.decay_row + h * a.decay_head;
      constexpr float LOG2E = 1.4426950408889634f;
      float later = 0.f;  // the decays of the chunks behind this one
      bool cut = false;   // and whether they hold a reset
#pragma unroll 1
      for (int i = 0; i < ADD_AHEAD; ++i) {
        if (i < n) fetch_decays(dec + i * C, decay, a.decay_token, chunk(i) * C, len);
        close_fetch();
      }
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int j = i + ADD_AHEAD;
        if (j < n) {
          if (!wait(&B.dec_empty[slot<ADD_RING>(j)], phase<ADD_RING>(j) + 1)) break;
          fetch_decays(dec + slot<ADD_RING>(j) * C, decay, a.decay_token, chunk(j) * C, len);
        }
        close_fetch();
        float2 g = fetched<ADD_AHEAD>(dec + slot<ADD_RING>(i) * C);
        const uint2 reset = take_resets(g);
        float down = g.x + g.y;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float y = __shfl_down_sync(0xffffffffu, down, o);
          if (lane + o < 32) down += y;
        }
        float after = __shfl_down_sync(0xffffffffu, down, 1);
        if (lane == 31) after = 0.f;
        after += later;
        float2 w = make_float2(fast_exp2((after + g.y) * LOG2E), fast_exp2(after * LOG2E));
        if (cut || (reset.x | reset.y)) {  // nothing of what came before a reset, unless it is NaN
          const uint32_t behind = ~0u << lane;
          if (cut || (reset.x & (behind << 1)) || (reset.y & behind)) w.x = 0.f * (after + g.y);
          if (cut || ((reset.x | reset.y) & (behind << 1))) w.y = 0.f * after;
          cut = true;
        }
        *reinterpret_cast<float2*>(dec + slot<ADD_RING>(i) * C + 2 * lane) = w;
        later += __shfl_sync(0xffffffffu, down, 0);
        arrive(&B.dec_full[slot<ADD_RING>(i)]);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (lane == 0) A.logs[(int64_t(b) * a.v_heads + h) * A.segments + seg] = cut ? later * 0.f - INFINITY : later;
    } else if (warp == LOAD_WARP) {
      if (elect_one()) {
        const uint32_t bytes = uint32_t(L::K_BYTES + (a.v_dim > 64 ? 2 : 1) * HALF);
        int i = 0;
#pragma unroll 1
        for (; i < n; ++i) {
          const int st = slot<ADD_STAGES>(i), t0 = chunk(i) * C;
          if (!wait.alone(&B.empty[st], phase<ADD_STAGES>(i) + 1)) break;
          uint8_t* stage = smem + st * L::STAGE;
          mbar_arrive_expect_tx(&B.full[st], bytes);
#pragma unroll 1
          for (int x = 0; x < DK; x += 64) tma_load(stage + x / 64 * HALF, &maps.k, x, hk, t0, b, &B.full[st]);
#pragma unroll 1
          for (int x = 0; x < a.v_dim; x += 64) tma_load(stage + L::K_BYTES + x / 64 * HALF, &maps.v, x, h, t0, b, &B.full[st]);
        }
        // copies in flight land before the block may end
#pragma unroll 1
        for (int k = max(0, i - ADD_STAGES); k < i; ++k)
          mbar_wait(&B.full[slot<ADD_STAGES>(k)], uint32_t(phase<ADD_STAGES>(k)) & 1, nullptr, 20000000LL);
      }
    } else if (warp == MMA_WARP) {
      const bool leader = elect_one();
      bool ok = tmem == 0;  // all 512 columns are this block's
      if (!ok) wait.stop();
#pragma unroll 1
      for (int i = 0; i < n && ok; ++i) {
        const int st = slot<ADD_STAGES>(i), run = i / ADD_RUN;
        if (i % ADD_RUN == 0 && !(ok = wait(&B.d_empty[run & 1], run / 2 + 1))) break;
        if (!(ok = wait(&B.full[st], phase<ADD_STAGES>(i), &B.kw_full[i & 1], i / 2))) break;
        fence_after();
        if (leader) {
          const uint64_t v = desc_mn(smem + st * L::STAGE + L::K_BYTES, HALF), kw = desc_mn(smem + L::KW + (i & 1) * 3 * L::K_BYTES, HALF);
          add_products<DK>((run & 1) * 128, v, kw, 0, i % ADD_RUN == 0);
          add_products<DK>((run & 1) * 128, v, kw, 1, false);
          commit(&B.kw_empty[i & 1]);
          commit(&B.empty[st]);
          if (i % ADD_RUN == ADD_RUN - 1 || i == n - 1) commit(&B.d_full[run & 1]);
        }
        __syncwarp();
      }
      if (leader) {
        commit(&B.done);  // every product issued has finished
        mbar_wait(&B.done, 0, nullptr, 20000000LL);
      }
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (tid == 0 && B.bail) record_error(A.err, SC_ERR_TIMEOUT);
  if (warp == MMA_WARP) tmem_free(tmem);
}

template <int DK>
__global__ void __launch_bounds__(THREADS, 1) chunk_kernel(const __grid_constant__ Args A, const __grid_constant__ Maps maps) {
  using L = Shape<DK>;
  extern __shared__ uint8_t raw[];
  // 1024-byte aligned, by an offset: through an integer the pointer would no longer be known to be shared memory's
  uint8_t* smem = raw + (0u - smem_u32(raw) & 1023u);
  Decays* dec = reinterpret_cast<Decays*>(smem + L::DEC);
  Bars& B = *reinterpret_cast<Bars*>(smem + L::BARS);
  const sc_linear& a = A.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int seg = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / (a.v_heads / a.k_heads);
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.tokens) : a.tokens;
  const int c0 = seg * A.per, all = (a.tokens + C - 1) / C, c1 = min(all, c0 + A.per);
  const int n = max(0, min(c1, (len + C - 1) / C) - c0);  // this segment's chunks with tokens
  if (tid == 0) {
    for (int i = 0; i < QS; ++i) mbar_init(&B.qk_full[0][i], 1), mbar_init(&B.qk_empty[0][i], 1);
    for (int i = 0; i < KS; ++i) mbar_init(&B.qk_full[1][i], 1), mbar_init(&B.qk_empty[1][i], 4 + 1);
    for (int i = 0; i < VS; ++i) mbar_init(&B.v_full[i], 1), mbar_init(&B.v_empty[i], 2);
    for (int i = 0; i < RING; ++i) mbar_init(&B.dec_full[i], 1), mbar_init(&B.dec_empty[i], 20);
    mbar_init(&B.a_full, 1), mbar_init(&B.a_empty, 4), mbar_init(&B.p_full, 4), mbar_init(&B.p_empty, 1);
    mbar_init(&B.o_full, 1), mbar_init(&B.o_empty, 4);
    for (int i = 0; i < 2; ++i) mbar_init(&B.kw_full[i], 4), mbar_init(&B.kw_empty[i], 1);
    mbar_init(&B.d_full, 1), mbar_init(&B.d_empty, 8), mbar_init(&B.s_full, 8), mbar_init(&B.s_empty, 1);
    mbar_init(&B.ends, 8), mbar_init(&B.outs, 4), mbar_init(&B.done, 2);
    B.bail = B.odd[0] = B.odd[1] = B.odd[2] = B.odd[3] = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) tmem_alloc(&B.tmem);
  if (a.v_dim <= 64) clear_halves(smem + L::V, VS, L::V_BYTES);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = B.tmem;
  const Waits wait{&B.bail};
  const uint32_t quarter = uint32_t(warp & 3) * 32, lanes = tmem + (quarter << 16);

  if (warp < STATE_WARP) {
    if (warp < OUT_WARP) {
      // ---- P
      fewer_registers<P_REGS>();
      const int g = lane >> 2, t = lane & 3, r0 = 16 * warp + g;
      uint8_t* p = smem + L::P;
      // the scale goes with the decays: 2^(G_i + log2 |scale| - G_j), its sign last
      const float shift = log2f(fabsf(a.scale));
      const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        if (!wait(&B.dec_full[slot<RING>(i)], phase<RING>(i), &B.a_full, i)) break;
        fence_after();
        const float* g2 = dec[slot<RING>(i)].g2;
        const float ga = g2[r0] + shift, gb = g2[r0 + 8] + shift;
        const bool cut = dec[slot<RING>(i)].resets != 0;
        bool ok = true;
#pragma unroll 1
        for (int c = 0; c < C; c += 32) {  // half the columns
          uint32_t r[16], pk[8], lo[8];
          ld_frag32(lanes + COL_A + c, r);
          wait_ld();
          if (c > 0) {
            fence_before();
            arrive(&B.a_empty);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int col = c + 8 * j + 2 * t;
            pk[2 * j] = pk[2 * j + 1] = lo[2 * j] = lo[2 * j + 1] = 0;
            if (c + 8 * j > 16 * warp + 15) continue;  // above the diagonal
            const float2 gj = *reinterpret_cast<const float2*>(g2 + col);
            float x0 = __uint_as_float(r[4 * j]) * fast_exp2(ga - gj.x), x1 = __uint_as_float(r[4 * j + 1]) * fast_exp2(ga - gj.y);
            float y0 = __uint_as_float(r[4 * j + 2]) * fast_exp2(gb - gj.x), y1 = __uint_as_float(r[4 * j + 3]) * fast_exp2(gb - gj.y);
            if (c + 8 * j + 7 > 16 * warp) {  // on it
              x0 = col <= r0 ? x0 : 0.f, x1 = col + 1 <= r0 ? x1 : 0.f;
              y0 = col <= r0 + 8 ? y0 : 0.f, y1 = col + 1 <= r0 + 8 ? y1 : 0.f;
            }
            if (cut) {  // what a reset parts
              const int fa = dec[slot<RING>(i)].from[r0], fb = dec[slot<RING>(i)].from[r0 + 8];
              x0 = col >= fa ? x0 : 0.f, x1 = col + 1 >= fa ? x1 : 0.f;
              y0 = col >= fb ? y0 : 0.f, y1 = col + 1 >= fb ? y1 : 0.f;
            }
            const float2 x = make_float2(x0, x1), y = make_float2(y0, y1);
            pk[2 * j] = rounded(x), pk[2 * j + 1] = rounded(y);
            lo[2 * j] = rounded(rest(x, pk[2 * j])) ^ sign, lo[2 * j + 1] = rounded(rest(y, pk[2 * j + 1])) ^ sign;
            pk[2 * j] ^= sign, pk[2 * j + 1] ^= sign;
          }
          if (c == 0 && !(ok = wait(&B.p_empty, i + 1))) break;
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // r0 and r0 + 8 have one place in the swizzle
            uint8_t* to = p + r0 * 128 + ((c / 8 + j ^ g) << 4) + 4 * t;
            *reinterpret_cast<uint32_t*>(to) = pk[2 * j];
            *reinterpret_cast<uint32_t*>(to + 8 * 128) = pk[2 * j + 1];
            *reinterpret_cast<uint32_t*>(to + HALF) = lo[2 * j];
            *reinterpret_cast<uint32_t*>(to + HALF + 8 * 128) = lo[2 * j + 1];
          }
        }
        if (!ok) break;
        arrive(&B.dec_empty[slot<RING>(i)]);
        fence_async();
        arrive(&B.p_full);
      }
    } else {
      // ---- the outputs
      fewer_registers<OUT_REGS>();
      const int t = lane & 3, ot = tid - OUT_WARP * 32;
      uint8_t* tile = smem + L::OUT;
      // where this lane's rows of transposed fragments go: token (lane / 16) 8 + lane % 8 of 16, pieces of 8 values
      const int token = (lane >> 4) * 8 + (lane & 7), piece = 4 * (warp & 3) + ((lane >> 3) & 1);
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const bool ok = wait(&B.dec_full[slot<RING>(i)], phase<RING>(i), &B.o_full, i);
        fence_after();
        if (ot == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        if (!out_all(ok)) break;  // and the tile's last store has read it
        const int t0 = (c0 + i) * C, m = len - t0;
        const float* eg = dec[slot<RING>(i)].eg;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {  // 16 value dimensions by 32 tokens at a time
          const int hf = q >> 1, j0 = 4 * (q & 1);
          uint32_t x[16], y[16];
          ld_frag32(lanes + (uint32_t(16 * hf) << 16) + col_x(i) + 8 * j0, x);
          ld_frag32(lanes + (uint32_t(16 * hf) << 16) + COL_I + 8 * j0, y);
          wait_ld();
          if (q == 3) {
            fence_before();
            arrive(&B.o_empty);
          }
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            uint32_t f[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int k = 4 * (j + e), col = 8 * (j0 + j + e) + 2 * t;
              const float2 s = *reinterpret_cast<const float2*>(eg + col);
              float2 o[2];
#pragma unroll
              for (int r = 0; r < 2; ++r)
                o[r] = __ffma2_rn(s, make_float2(__uint_as_float(x[k + 2 * r]), __uint_as_float(x[k + 2 * r + 1])),
                                  make_float2(__uint_as_float(y[k + 2 * r]), __uint_as_float(y[k + 2 * r + 1])));
              if (m < C) {  // zeros past the length
                if (col >= m) o[0].x = o[1].x = 0.f;
                if (col + 1 >= m) o[0].y = o[1].y = 0.f;
              }
              f[2 * e] = rounded(o[0]);
              f[2 * e + 1] = rounded(o[1]);
            }
            const int row = 8 * (j0 + j) + token, pc = piece + 2 * hf;
            store_transposed(smem_u32(tile) + (pc >> 3) * HALF + row * 128 + (((pc & 7) ^ (row & 7)) << 4), f[0], f[1], f[2], f[3]);
          }
        }
        arrive(&B.dec_empty[slot<RING>(i)]);
        fence_async();
        out_sync();
        if (ot == 0) {
          tma_store(&maps.out, tile, 0, h, t0, b);
          if (a.v_dim > 64) tma_store(&maps.out, tile + HALF, 64, h, t0, b);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
      // zeros past the last chunk with tokens, 16 bytes at a time
      const int t1 = (c0 + n) * C, pieces = a.v_dim / 8, rows = max(0, min(a.tokens, c1 * C) - t1);
#pragma unroll 1
      for (int e = ot; e < rows * pieces; e += 128)
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) +
                                  ((int64_t(b) * a.tokens + t1 + e / pieces) * a.v_heads + h) * a.v_dim + 8 * (e % pieces)) =
            make_uint4(0, 0, 0, 0);
      if (ot == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      out_sync();
      if (n > 0 && wait(&B.ends, 0) && B.odd[warp & 3] && !*wait.bail)
        mend_outputs<DK>(A, smem + L::Q, smem + L::P, int(quarter) + lane, c0 * C, min(len, (c0 + n) * C));
      arrive(&B.outs);
    }
  } else if (warp < KW_WARP) {
    // ---- the state: value dimension `dv`, key dimensions k0 .. k0 + DK / 2 - 1
    constexpr int N = DK / 2;
    more_registers<STATE_REGS>();
    const int dv = int(quarter) + lane, k0 = (warp - STATE_WARP) / 4 * N;
    float2 S[N / 2];
    const int64_t head = int64_t(b) * a.v_heads + h;
    const bool started = A.segments > 1, there = started || (a.state_in && dv < a.v_dim);
    if (started) pdl_wait();  // for the states before the segments: only these warps read them
    const float* from = started ? A.parts + ((head * A.segments + seg) * DK + k0) * 128 + dv
                                : a.state_in + (head * a.k_dim + k0) * a.v_dim + dv;
    const int kd = started ? DK : a.k_dim, ld = started ? 128 : a.v_dim;
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      S[k].x = there && k0 + 2 * k < kd ? *from : 0.f;
      from += ld;
      S[k].y = there && k0 + 2 * k + 1 < kd ? *from : 0.f;
      from += ld;
    }
    // S^T as two terms, the A operand of X. The first 16 are made while the last X still reads the old ones (one prompt
    // of 32768 tokens of 16 heads: 183.7 us, with none 185.4, with half of them 184.4)
    auto terms = [&](int k, uint32_t (&hi)[8], uint32_t (&lo)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        hi[e] = rounded(S[k / 2 + e]);
        lo[e] = rounded(rest(S[k / 2 + e], hi[e]));
      }
    };
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      uint32_t hi[8], lo[8];
      terms(0, hi, lo);
      if (i > 0) {
        if (!wait(&B.s_empty, i - 1)) break;
        fence_after();
      }
#pragma unroll
      for (int k = 0; k < N; k += 16) {
        if (k > 0) terms(k, hi, lo);
        st8(lanes + COL_S + (k0 + k) / 2, hi);
        st8(lanes + COL_S + DK / 2 + (k0 + k) / 2, lo);
      }
      wait_st();
      fence_before();
      arrive(&B.s_full);
      if (!wait(&B.dec_full[slot<RING>(i)], phase<RING>(i), &B.d_full, i)) break;
      fence_after();
      const float2 d = make_float2(dec[slot<RING>(i)].a, dec[slot<RING>(i)].a), one = make_float2(dec[slot<RING>(i)].one, dec[slot<RING>(i)].one);
#pragma unroll
      for (int k = 0; k < N; k += 16) {
        uint32_t r[16];
        ld16(lanes + COL_D + k0 + k, r);
        wait_ld();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float2& x = S[k / 2 + e];
          x = __ffma2_rn(d, x, __ffma2_rn(one, x, make_float2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]))));
        }
      }
      fence_before();
      arrive(&B.d_empty);
      arrive(&B.dec_empty[slot<RING>(i)]);
    }
    float2 zero = make_float2(0.f, 0.f);  // NaN where a state is not finite
#pragma unroll
    for (int k = 0; k < N / 2; ++k) zero = __ffma2_rn(S[k], make_float2(0.f, 0.f), zero);
    if (__any_sync(0xffffffffu, !(zero.x + zero.y == 0.f))) B.odd[warp & 3] = 1;
    arrive(&B.ends);
    if (seg == A.segments - 1) {
      // in place: the outputs may go back to the state before
      if (A.segments == 1 && a.state_in == a.state_out) wait(&B.outs, 0);
      float* to = a.state_out + (head * a.k_dim + k0) * a.v_dim + dv;
      const int kd = dv < a.v_dim ? a.k_dim - k0 : 0;
#pragma unroll
      for (int k = 0; k < N / 2; ++k) {
        if (2 * k < kd) *to = S[k].x;
        to += a.v_dim;
        if (2 * k + 1 < kd) *to = S[k].y;
        to += a.v_dim;
      }
    }
  } else if (warp < MMA_WARP) {
    // ---- w K
    fewer_registers<KW_REGS>();
    const int lt = tid - KW_WARP * 32;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int m = len - (c0 + i) * C;
      if (!wait(&B.dec_full[slot<RING>(i)], phase<RING>(i), &B.qk_full[1][slot<KS>(i)], phase<KS>(i))) break;
      const uint8_t* k = smem + L::K + slot<KS>(i) * L::K_BYTES;
      const float* w = dec[slot<RING>(i)].w;
      if (m < C) {
        if (!wait(&B.v_full[slot<VS>(i)], phase<VS>(i))) break;
        clear_values(smem + L::V + slot<VS>(i) * L::V_BYTES, m, lt, 128);
      }
      bool ok = true;
#pragma unroll 1
      for (int hf = 0; hf < 2; ++hf) {
        if (!(ok = wait(&B.kw_empty[hf], i + 1))) break;
#pragma unroll 1
        for (int j = lt; j < C / 2 * DK / 8; j += 128) {
          const int r = C / 2 * hf + j / 8 % (C / 2), at = j / (C / 2 * 8) * HALF + r * 128 + j % 8 * 16;
          split_piece(k + at, w[r], r < m, smem + L::KW + at, L::K_BYTES);
        }
        fence_async();
        arrive(&B.kw_full[hf]);
      }
      if (!ok) break;
      arrive(&B.qk_empty[1][slot<KS>(i)]);
      arrive(&B.dec_empty[slot<RING>(i)]);
    }
  } else {
    fewer_registers<CONTROL_REGS>();
    if (warp == DECAY_WARP) {
      // ---- a chunk's decays: a lane tokens 2 lane and 2 lane + 1, sums from the front and from the back
      const float* decay = a.decay + b * a.decay_row + h * a.decay_head;
      float* got = reinterpret_cast<float*>(smem + L::RAW);
#pragma unroll 1
      for (int i = 0; i < AHEAD; ++i) {
        if (i < n) fetch_decays(got + i * C, decay, a.decay_token, (c0 + i) * C, len);
        close_fetch();
      }
      auto decays = [&](int i) -> bool {
        float2 g = fetched<AHEAD - 1>(got + slot<AHEAD>(i) * C);
        const uint2 reset = take_resets(g);
        const float g0 = g.x, g1 = g.y, pair = g0 + g1;
        if (i + AHEAD < n) fetch_decays(got + slot<AHEAD>(i) * C, decay, a.decay_token, (c0 + i + AHEAD) * C, len);
        close_fetch();
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
        Decays& D = dec[slot<RING>(i)];
        if (!wait(&B.dec_empty[slot<RING>(i)], phase<RING>(i) + 1)) return false;
        float2 eg = make_float2(fast_exp2(e0) * a.scale, fast_exp2(e1) * a.scale);
        float2 w = make_float2(fast_exp2((after + g1) * LOG2E), fast_exp2(after * LOG2E));
        const bool cut = (reset.x | reset.y) != 0;
        if (cut) {  // zeros across a reset, unless a NaN is in the sum
          const uint32_t behind = ~0u << lane, upto = ~(behind << 1), x = reset.x & upto, y = reset.y & ~behind;
          const uint32_t y1 = reset.y & upto;
          // tokens 2 lane and 2 lane + 1: the last reset at or before them (an empty mask gives -2 or -1)
          D.from[2 * lane] = uint8_t(max(0, max(62 - 2 * __clz(x), 63 - 2 * __clz(y))));
          D.from[2 * lane + 1] = uint8_t(max(0, max(62 - 2 * __clz(x), 63 - 2 * __clz(y1))));
          if (x | y) eg.x = 0.f * e0;
          if (x | y1) eg.y = 0.f * e1;
          if ((reset.x & (behind << 1)) | (reset.y & behind)) w.x = 0.f * (after + g1);
          if ((reset.x | reset.y) & (behind << 1)) w.y = 0.f * after;
        }
        *reinterpret_cast<float2*>(&D.g2[2 * lane]) = make_float2(e0, e1);
        *reinterpret_cast<float2*>(&D.eg[2 * lane]) = eg;
        *reinterpret_cast<float2*>(&D.w[2 * lane]) = w;
        if (lane == 31) {
          const bool near = fabsf(up) < 0.69314718f;  // past it, growth included, a itself
          D.a = cut ? 0.f * up : near ? expm1_near(up) : expf(up), D.one = near && !cut ? 1.f : 0.f;
          D.resets = cut;
        }
        arrive(&B.dec_full[slot<RING>(i)]);
        return true;
      };
      const bool leader = elect_one();
      int i = -1;  // the decays a chunk ahead of the values
#pragma unroll 1
      for (; i < n; ++i) {
        if (i + 1 < n && !decays(i + 1)) break;
        if (i < 0) continue;
        if (!wait(&B.v_empty[slot<VS>(i)], phase<VS>(i) + 1)) break;
        if (leader) {
          mbar_arrive_expect_tx(&B.v_full[slot<VS>(i)], (a.v_dim > 64 ? 2 : 1) * HALF);
#pragma unroll 1
          for (int x = 0; x < a.v_dim; x += 64)
            tma_load(smem + L::V + slot<VS>(i) * L::V_BYTES + x / 64 * HALF, &maps.v, x, h, (c0 + i) * C, b, &B.v_full[slot<VS>(i)]);
        }
        __syncwarp();
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (leader)  // copies in flight land before the block may end
#pragma unroll 1
        for (int k = max(0, i - VS); k < i; ++k) mbar_wait(&B.v_full[slot<VS>(k)], uint32_t(phase<VS>(k)) & 1, nullptr, 20000000LL);
      __syncwarp();
    } else if (warp == LOAD_WARP) {
      // ---- keys and queries
      if (elect_one()) {
        static_assert(QS == KS && L::K == L::Q + QS * L::K_BYTES, "queries' and keys' places");
        int e = 0;
#pragma unroll 1
        for (; e < 2 * n; ++e) {  // by turns
          const int i = e >> 1, of = 1 - (e & 1), st = slot<KS>(i);
          if (!wait.alone(&B.qk_empty[of][st], phase<KS>(i) + 1)) break;
          mbar_arrive_expect_tx(&B.qk_full[of][st], L::K_BYTES);
#pragma unroll 1
          for (int x = 0; x < DK; x += 64)
            tma_load(smem + L::Q + (of * QS + st) * L::K_BYTES + x / 64 * HALF, of ? &maps.k : &maps.q, x, hk, (c0 + i) * C, b, &B.qk_full[of][st]);
        }
        // copies in flight land before the block may end
#pragma unroll 1
        for (int k = max(0, e - 2 * KS); k < e; ++k)
          mbar_wait(&B.qk_full[1 - (k & 1)][slot<KS>(k >> 1)], uint32_t(phase<KS>(k >> 1)) & 1, nullptr, 20000000LL);
      }
      __syncwarp();
    } else if (warp == SUM_WARP) {
      // ---- D
      const bool leader = elect_one();
      const uint64_t kw = desc_mn(smem + L::KW, HALF);
#pragma unroll 1
      for (int i = 0; i < n && tmem == 0; ++i) {
        const uint64_t vt = desc_mn(smem + L::V + slot<VS>(i) * L::V_BYTES, HALF);
        bool ok = true;
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) {
          if (!(ok = wait(&B.v_full[slot<VS>(i)], phase<VS>(i), &B.d_empty, i + 1, &B.kw_full[hf], i))) break;
          fence_after();
          if (leader) {
            add_products<DK>(COL_D, vt, kw, hf, hf == 0);
            commit(&B.kw_empty[hf]);
            if (hf > 0) {
              commit(&B.d_full);
              commit(&B.v_empty[slot<VS>(i)]);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
      }
      if (leader) commit(&B.done);
      __syncwarp();
    } else if (warp == MMA_WARP) {
      // ---- the products. The whole warp follows the loop, so that what a product is given is uniform; one lane issues.
      // All 512 columns are this block's, so tensor memory starts at address 0.
      const bool leader = elect_one();
      auto a_product = [&](int i) {
        const uint8_t *q = smem + L::Q + slot<QS>(i) * L::K_BYTES, *k = smem + L::K + slot<KS>(i) * L::K_BYTES;
        if (leader) {
          uint64_t qd = desc_k(q), kd = desc_k(k);
#pragma unroll 1
          for (int x = 0; x < DK / 64; ++x, qd += HALF >> 4, kd += HALF >> 4)
#pragma unroll
            for (int s = 0; s < 4; ++s) mma_ss(COL_A, qd + 2 * s, kd + 2 * s, idesc_bf16(64, 64, false, false), x > 0 || s > 0);
          commit(&B.a_full);
          commit(&B.qk_empty[1][slot<KS>(i)]);
        }
        __syncwarp();
      };
      bool ok = tmem == 0;
      if (!ok) wait.stop();
#pragma unroll 1
      for (int i = -1; i < n && ok; ++i) {
        const uint64_t vt = desc_mn(smem + L::V + slot<VS>(i) * L::V_BYTES, HALF);
        if (i + 1 < n) {  // ahead: P of the next chunk is made while this chunk's products run
          const int j = i + 1;
          if (!(ok = wait(&B.qk_full[0][slot<QS>(j)], phase<QS>(j), &B.qk_full[1][slot<KS>(j)], phase<KS>(j), &B.a_empty, i))) break;
          fence_after();
          a_product(j);
        }
        if (i >= 0) {
          if (!(ok = wait(&B.s_full, i))) break;
          fence_after();
          if (leader) {
            const uint64_t qd = desc_k(smem + L::Q + slot<QS>(i) * L::K_BYTES);
#pragma unroll 1
            for (int e = 2 * (DK / 64) - 1; e >= 0; --e) {  // the rest, then the rounded state; 64 key dimensions each
              const int x = e % (DK / 64);
#pragma unroll
              for (int s = 0; s < 4; ++s)
                mma_ts(col_x(i), COL_S + 32 * e + 8 * s, qd + uint32_t(x * (HALF >> 4) + 2 * s), idesc_bf16(128, 64, false, false),
                       e < 2 * (DK / 64) - 1 || s > 0);
            }
            commit(&B.s_empty);
            commit(&B.qk_empty[0][slot<QS>(i)]);
          }
          __syncwarp();
        }
        if (i < 0) continue;
        if (!(ok = wait(&B.p_full, i, &B.v_full[slot<VS>(i)], phase<VS>(i), &B.o_empty, i + 1))) break;
        if (len - (c0 + i) * C < C && !(ok = wait(&B.kw_full[0], i))) break;  // the last chunk's values are cleared
        fence_after();
        if (leader) {
          uint64_t pd = desc_k(smem + L::P + HALF);
#pragma unroll 1
          for (int term = 1; term >= 0; --term, pd -= HALF >> 4)  // the rest, then the rounded
#pragma unroll
            for (int s = 0; s < C / 16; ++s)
              mma_ss(COL_I, vt + 128 * s, pd + 2 * s, idesc_bf16(128, 64, true, false), term < 1 || s > 0);
          commit(&B.o_full);
          commit(&B.p_empty);
          commit(&B.v_empty[slot<VS>(i)]);
        }
        __syncwarp();
      }
      if (leader) {
        commit(&B.done);  // every product issued has finished
        mbar_wait(&B.done, 0, nullptr, 20000000LL);
      }
      __syncwarp();
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (tid == 0 && B.bail) record_error(A.err, SC_ERR_TIMEOUT);
  if (warp == MMA_WARP) tmem_free(tmem);
}

// the states before the segments, in place of what the segments add: a thread a value
template <int DK>
__global__ void __launch_bounds__(256) scan_kernel(const Args A) {
  const sc_linear& a = A.a;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t head = blockIdx.x;
  const int e = blockIdx.y * 256 + threadIdx.x, k = e / 128, dv = e % 128;
  float* part = A.parts + head * A.segments * DK * 128 + e;
  float S = a.state_in && k < a.k_dim && dv < a.v_dim ? a.state_in[(head * a.k_dim + k) * a.v_dim + dv] : 0.f;
  const int last = A.segments - 1;
  for (int s0 = 0; s0 < last; s0 += 8) {
    float log[8], add[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (s0 + i < last) log[i] = A.logs[head * A.segments + s0 + i], add[i] = part[int64_t(s0 + i) * DK * 128];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (s0 + i < last) {
        part[int64_t(s0 + i) * DK * 128] = S;
        S = log[i] > -0.69314718f ? fmaf(expm1f(log[i]), S, S + add[i]) : fmaf(expf(log[i]), S, add[i]);
      }
  }
  part[int64_t(last) * DK * 128] = S;
}

// The segments that cost least, in chunks' time of an SM: waves of blocks times a segment's chunks (and about three
// to start and end a block), the first launch's at three fifths, and the scan over the segments' states. Measured with 16
// heads of one sequence: 512 tokens 18.8 us in four segments, 21.0 in one; 1024 20.4 in eight, 36.3 in one; 32768 174 in
// nine, 355 in four, 192 in 18 (a second wave). 96 heads of 1536 tokens: 53 in one, 82 in two.
inline int segments_of(const sc_linear& a) {
  const int64_t heads = int64_t(a.batch) * a.v_heads;
  const int chunks = int(ceil_div(a.tokens, C));
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= std::max(1, std::min(chunks / 2, SMS)); ++s) {
    const double per = double(ceil_div(chunks, s)) + 3;
    double cost = double(ceil_div(heads * s, SMS)) * per;
    if (s > 1) cost += 0.6 * double(ceil_div(heads * (s - 1), SMS)) * per + 1 + 0.02 * double(heads * s);
    if (cost < least) least = cost, best = s;
  }
  return best;
}

inline size_t parts_bytes(const sc_linear& a, int segments) {
  const int dk = a.k_dim <= 64 ? 64 : 128;
  return segments > 1 ? size_t(a.batch) * a.v_heads * segments * (size_t(dk) * 128 + 4) * 4 : 0;
}

size_t workspace(const sc_linear& a) { return parts_bytes(a, segments_of(a)); }

// a tensor of (batch, tokens, heads, dim) as a map; the strides of axes of one entry are not looked at
inline int map_of(CUtensorMap* m, const void* p, int dim, int heads, int tokens, int batch, int64_t head, int64_t token, int64_t row) {
  const cuuint64_t dims[4] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(tokens), cuuint64_t(batch)};
  const cuuint64_t any = cuuint64_t(dim) * 2;
  const cuuint64_t strides[3] = {heads > 1 ? cuuint64_t(head) * 2 : any, tokens > 1 ? cuuint64_t(token) * 2 : any,
                                 batch > 1 ? cuuint64_t(row) * 2 : any};
  const cuuint32_t box[4] = {64, 1, C, 1}, each[4] = {1, 1, 1, 1};
  const EncodeTiled encode = encode_tiled();
  return encode && encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, box, each,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? SC_OK
             : SC_ERR_CUDA;
}

template <int DK>
int run(const Args& A, cudaStream_t s) {
  const sc_linear& a = A.a;
  Maps maps;
  const int64_t token = int64_t(a.v_heads) * a.v_dim;
  if (map_of(&maps.q, a.q, a.k_dim, a.k_heads, a.tokens, a.batch, a.q_head, a.q_token, a.q_row) ||
      map_of(&maps.k, a.k, a.k_dim, a.k_heads, a.tokens, a.batch, a.k_head, a.k_token, a.k_row) ||
      map_of(&maps.v, a.v, a.v_dim, a.v_heads, a.tokens, a.batch, a.v_head, a.v_token, a.v_row) ||
      map_of(&maps.out, a.out, a.v_dim, a.v_heads, a.tokens, a.batch, a.v_dim, token, token * a.tokens))
    return cuda_failed(cudaErrorInvalidValue, "linear attention tensor map");
  const dim3 grid(unsigned(A.segments), unsigned(a.v_heads), unsigned(a.batch));
  constexpr int smem = Shape<DK>::BYTES;
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  if (int rc = raise_smem(reinterpret_cast<const void*>(chunk_kernel<DK>), smem, "linear attention smem attribute"))
    return rc;
  if (A.segments > 1) {
    constexpr int add_smem = AddShape<DK>::BYTES;
    static_assert(add_smem <= 227 * 1024, "shared memory of a block");
    if (int rc = raise_smem(reinterpret_cast<const void*>(add_kernel<DK>), add_smem, "linear attention smem attribute"))
      return rc;
    add_kernel<DK><<<dim3(grid.x - 1, grid.y, grid.z), THREADS, add_smem, s>>>(A, maps);
    // the scan and the whole as programmatic dependents: their blocks start as the ones before leave their SMs
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(a.batch) * unsigned(a.v_heads), DK * 128 / 256);
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, scan_kernel<DK>, A)) return cuda_failed(e, "linear attention scan launch");
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, chunk_kernel<DK>, A, maps)) return cuda_failed(e, "linear attention launch");
  } else {
    chunk_kernel<DK><<<grid, THREADS, smem, s>>>(A, maps);
  }
  if (cudaError_t e = cudaGetLastError()) return cuda_failed(e, "linear attention launch");
  return SC_OK;
}

// a map takes no stride of zero (a broadcast axis) and none past 2^40 bytes
bool takes(const sc_linear& a) {
  auto fits = [&](int n, int64_t stride) { return n < 2 || (stride > 0 && stride < (int64_t(1) << 38)); };
  return a.dtype == SC_BF16 && a.tokens > 0 && fits(a.k_heads, a.q_head) && fits(a.k_heads, a.k_head) &&
         fits(a.v_heads, a.v_head) && fits(a.tokens, a.q_token) && fits(a.tokens, a.k_token) && fits(a.tokens, a.v_token) &&
         fits(a.batch, a.q_row) && fits(a.batch, a.k_row) && fits(a.batch, a.v_row);
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
