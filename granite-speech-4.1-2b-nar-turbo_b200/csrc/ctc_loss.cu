// Connectionist temporal classification loss (Graves, Fernandez, Gomez, Schmidhuber, ICML 2006) of the encoder's CTC
// heads, and its gradient with respect to the logits.
//
//   p_t = softmax(logits[t]);  l' = blank l1 blank l2 ... blank, 2 S + 1 states
//   alpha_t(s) = p_t(l'_s) (alpha_{t-1}(s) + alpha_{t-1}(s-1) + [l'_s != blank, l'_s != l'_{s-2}] alpha_{t-1}(s-2))
//   Z = alpha_{n-1}(2S) + alpha_{n-1}(2S-1), loss = -log Z, beta the same from the end (without the emission at t)
//   dlogits[t, v] = dloss (p_t(v) - sum over s with l'_s = v of alpha_t(s) beta_t(s) / Z), 0 for t >= n
//
// Three launches: rows (maximum and sum of exponentials of every frame, the emissions of blank and labels; HBM-bound),
// lattice (both chains, the posteriors; a chain of n dependent steps), gradient (HBM-bound).  The emissions are taken
// against the frame's largest logit, so the frame's normaliser stays out of the chain: it cancels in the posteriors,
// and the loss adds the normalisers in 64 bits.
#include <limits.h>

#include <type_traits>

#include "gsn_kernels.cuh"
#include "gsn_ptx.cuh"

namespace gsn {

namespace ctc_loss_impl {

using rows_impl::from_f32;
using rows_impl::to_f32;

constexpr float kLog2e = 1.4426950408889634f;

// ---- numbers of the lattice ------------------------------------------------------------------------------------------
// A state is m * 2^e with its own integer exponent.  Sums over paths leave fp32's range within a few dozen frames, and
// a state thousands of octaves below its frame's largest can still carry the whole posterior (a confident model and
// another transcript), so neither fp32 with a scale a frame nor fp64 holds them; the logarithm in fp32 would lose
// 2^-12 at -4000.  m lies within a few octaves of 1; a zero has e near kZeroExp, so that its terms vanish in any sum.
//   bounds: a frame's emission is 2^-15870 at the least or impossible, kMaxCtcFrames of them stay above -2^28;
//   kZeroExp = -2^29, e is held at or above it, and no sum of three exponents leaves an int.
constexpr int kZeroExp = -(1 << 29);
constexpr int kZeroBelow = -(1 << 28);        // exponents below it are zeros

// 2^d for d <= 127 (0 from -127 down)
__device__ __forceinline__ float pow2i(int d) { return __int_as_float(max(d + 127, 0) << 23); }

// Stored numbers, emissions and states alike, are the high word of an fp64: 11 bits of exponent, 20 of mantissa,
// rounded to nearest (2^-21, an eighth of an fp32 logit's own step at 10).  0 is zero.  An emission is against the
// frame's likeliest class of the transcript; a state against its lane's reference exponent, stored beside it.  That
// holds states down to 2^-kWordSpan of their lane's largest.  Labels that the logits favour in another order than the
// transcript's lie further apart, and the lower one can carry the whole posterior: such an utterance is walked again
// with every state's own exponent stored.
constexpr uint32_t kWordOne = 1u << 20;       // words below it are zeros
constexpr int kWordSpan = 1000;
__device__ __forceinline__ uint32_t to_word(float m, int e) {          // m * 2^e, 0 where it leaves the range
  const uint32_t v = ((__float_as_uint(m) + 4u) >> 3) + ((uint32_t)(e + 896) << 20);
  return e < -kWordSpan ? 0u : v;
}
// A state with its own exponent: 20 bits of mantissa and the low 12 of the exponent, its upper 16 apart (0: a zero).
constexpr int kWideBias = (1 << 28) - (1 << 16);   // exponents from -2^28 + 2^16 to 2^16 as 28 bits
__device__ __forceinline__ uint32_t to_wide(float m, int e, uint32_t& upper) {
  const uint32_t bits = __float_as_uint(m), t = ((bits & 0x7FFFFFu) + 4u) >> 3;
  const int field = e < kZeroBelow ? 0 : e + (int)(bits >> 23) - 127 + (int)(t >> 20) + kWideBias;
  upper = (uint32_t)field >> 12;
  return (t << 12) | ((uint32_t)field & 0xFFFu);
}
__device__ __forceinline__ float wide_mantissa(uint32_t v) { return __uint_as_float((v >> 12 << 3) | 0x3F800000u); }
__device__ __forceinline__ int wide_exponent(uint32_t v, uint32_t upper) {
  return (int)((upper << 12) | (v & 0xFFFu)) - kWideBias;
}
// A double in [0, 2^127) cut to fp32, zero below 2^-126: three integer instructions (the conversion instruction from
// fp64 runs at a sixteenth of their rate or less: with it a frame of three pairs a lane took 455 cycles, not 160).
__device__ __forceinline__ float to_float(double d) {
  const uint32_t hi = (uint32_t)__double2hiint(d), lo = (uint32_t)__double2loint(d);
  return hi < (897u << 20) ? 0.f : __uint_as_float(__funnelshift_l(lo, hi - (896u << 20), 3));
}
__device__ __forceinline__ float word_mantissa(uint32_t v) {
  return __uint_as_float(((v & (kWordOne - 1)) << 3) | 0x3F800000u);
}

// ---- vectors of eight logits at any alignment ------------------------------------------------------------------------
// Elements before the first 16-byte boundary of a row, which the vector loops leave to single loads.
template <typename T>
__device__ __forceinline__ int head_of(const T* row, int V) {
  const int h = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
  return h < V ? h : V;
}

// ---- rows ------------------------------------------------------------------------------------------------------------
struct Online {                                  // running maximum and sum of exponentials against it
  float top, sum;
};

__device__ __forceinline__ void online_one(Online& o, float x) {
  if (x > o.top) {
    o.sum *= ex2_approx((o.top - x) * kLog2e);
    o.top = x;
  }
  o.sum += x == -INFINITY ? 0.f : ex2_approx((x - o.top) * kLog2e);
}

// eight at a time: a branch where the maximum moves, pairs for the rest
__device__ __forceinline__ void online_eight(Online& o, const float2 (&f)[4]) {
  using rows_impl::add2;
  using rows_impl::both;
  using rows_impl::mul2;
  const float top = fmaxf(fmaxf(fmaxf(f[0].x, f[0].y), fmaxf(f[1].x, f[1].y)),
                          fmaxf(fmaxf(f[2].x, f[2].y), fmaxf(f[3].x, f[3].y)));
  if (top > o.top) {
    o.sum *= ex2_approx((o.top - top) * kLog2e);
    o.top = top;
  }
  const float2 minus = both(o.top == -INFINITY ? 0.f : -o.top);
  float2 e[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 d = mul2(add2(f[k], minus), both(kLog2e));
    e[k] = make_float2(ex2_approx(d.x), ex2_approx(d.y));
  }
  const float2 s = add2(add2(e[0], e[1]), add2(e[2], e[3]));
  o.sum += s.x + s.y;
}

__device__ __forceinline__ Online online_join(Online a, Online b) {
  const float top = fmaxf(a.top, b.top);
  if (top == -INFINITY) return Online{top, a.sum + b.sum};     // nothing seen, or NaN
  return Online{top, a.sum * ex2_approx((a.top - top) * kLog2e) + b.sum * ex2_approx((b.top - top) * kLog2e)};
}

template <typename T, int THREADS>
__device__ __forceinline__ Online scan_row(const T* __restrict__ x, int V, int tid) {
  Online o{-INFINITY, 0.f};
  const int head = head_of(x, V), vecs = (V - head) / 8;
  if (tid < head) online_one(o, to_f32(x[tid]));
  const T* body = x + head;
  int i = tid;
  for (; i + 3 * THREADS < vecs; i += 4 * THREADS) {           // four loads under way at once
    rows_impl::Vec8<T> r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int q = 0; q < rows_impl::Vec8<T>::Q; ++q)
        r[u].q[q] = __ldg(reinterpret_cast<const uint4*>(body + (int64_t)(i + u * THREADS) * 8) + q);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float2 f[4];
      rows_impl::unpack(r[u], f);
      online_eight(o, f);
    }
  }
  for (; i < vecs; i += THREADS) {
    rows_impl::Vec8<T> r;
#pragma unroll
    for (int q = 0; q < rows_impl::Vec8<T>::Q; ++q)
      r.q[q] = __ldg(reinterpret_cast<const uint4*>(body + (int64_t)i * 8) + q);
    float2 f[4];
    rows_impl::unpack(r, f);
    online_eight(o, f);
  }
  for (int v = head + vecs * 8 + tid; v < V; v += THREADS) online_one(o, to_f32(x[v]));
  // one rescaling to the warp's largest, then plain sums
  float top = o.top;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float sum = o.top == top ? o.sum : o.top == -INFINITY ? o.sum : o.sum * ex2_approx((o.top - top) * kLog2e);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  return Online{top, sum};
}

// The transcript's places in the order of their labels (the blank's own place, number S, among them), so that the
// gradient adds the posteriors of one class next to one another; and whether any label lies outside the vocabulary.
__device__ __forceinline__ void plan_utterance(const CtcArgs& a, int b) {
  const int len = __ldg(a.target_lengths + b);
  const bool fits = len >= 0 && len <= a.S;
  const int* targets = a.targets + (int64_t)b * a.S;
  int2* order = a.order + (int64_t)b * a.pitch;
  int bad = !fits;
  const int count = fits ? len + 1 : 0;          // entry len: the blank
  __shared__ int labels[kMaxCtcLabels + 1];
  for (int i = threadIdx.x; i < count; i += blockDim.x) labels[i] = i < len ? __ldg(targets + i) : a.blank;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    const int v = labels[i];
    bad |= v < 0 || v >= a.V;
    int rank = 0;
    for (int j = 0; j < i; ++j) rank += labels[j] <= v;
    for (int j = i + 1; j < count; ++j) rank += labels[j] < v;
    order[rank] = make_int2(i < len ? i : a.S + 1, v);           // where its posterior lies, its class
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) {
    a.bad[b] = bad;
    a.again[b] = 0;
    a.raw_loss[b] = a.loss[b] = NAN;               // what stays where a wait of the lattice runs out
  }
}

// exp(a) as a stored word, for a <= 0; 0 below kLowest and for NaN (the frame's sum tells of it)
constexpr float kLowest = -690.f;
// A frame with a class of the transcript below kLowest and not below kImpossible has words of 14 bits of exponent and 18
// of mantissa, and its span is marked: beyond any block's kFastSpan, so the lattice comes upon it among its slow frames.
constexpr float kImpossible = -11000.f;
constexpr int kFarShift = 18, kFarBias = 15872;
constexpr uint32_t kFarSpan = 1u << 16;
__device__ __forceinline__ uint32_t far_emission_word(float logit, float best) {
  const double d = (double)logit - (double)best, a = d * 1.4426950408889634, r = rint(a);
  if (!(d >= (double)kImpossible)) return 0u;
  return ((__float_as_uint(ex2_approx((float)(a - r))) + 16u) >> 5) + ((uint32_t)((int)r + kFarBias - 127) << kFarShift);
}
template <typename T>
__device__ __noinline__ void write_far_emissions(const T* x, uint32_t* em, const int* targets, int len, int S, int blank,
                                                 int V, float best, int lane) {
  __syncwarp();                                    // behind the frame's other words
  for (int i = lane; i <= len; i += 32) {
    const int v = i < len ? __ldg(targets + i) : blank;
    em[i < len ? i : S + 1] = v < 0 || v >= V ? 0u : far_emission_word(to_f32(x[v]), best);
  }
}

__device__ __forceinline__ uint32_t emission_word(float a) {
  const float r = fmaf(a, kLog2e, 12582912.f);   // 1.5 * 2^23: the nearest integer of a / ln 2 in the low bits
  const float f = fmaf(a, kLog2e, 12582912.f - r);
  const uint32_t v = ((__float_as_uint(ex2_approx(f)) + 4u) >> 3) + (__float_as_uint(r) << 20) + (896u << 20);
  return a >= kLowest ? v : 0u;
}

// Emission words of F frames that follow one another (frame, x: of the first; count <= F of them are there): labels at
// [0, len), a zero at S, the blank at S + 1, and at S + 2 how many octaves the least of them lies below the likeliest
// (with kFarSpan where that takes the other words).
// best[f]: the likeliest one's logit.  One warp; a label is looked up once for all its frames, and the first 32 KEEP
// labels' logits stay in registers between the two passes.
template <typename T, int F, int KEEP>
__device__ __forceinline__ void write_emissions(const CtcArgs& a, const T* x, int64_t frame, int count, int b, int lane,
                                                float (&best)[F]) {
  uint32_t* em = reinterpret_cast<uint32_t*>(a.post) + frame * a.pitch;
  const int len = min(max(__ldg(a.target_lengths + b), 0), a.S);
  const int* targets = a.targets + (int64_t)b * a.S;
  auto label = [&](int i) {
    const int v = i < len ? __ldg(targets + i) : a.blank;
    return v < 0 || v >= a.V ? -1 : v;
  };
  auto logit = [&](int v, int f) { return v < 0 || f >= count ? -INFINITY : to_f32(x[f * a.ld_t + v]); };
  float kept[KEEP][F], least[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    best[f] = logit(a.blank, f);
    least[f] = 0.f;
  }
#pragma unroll
  for (int u = 0; u < KEEP; ++u)
    if (u * 32 < len) {
      const int v = u * 32 + lane < len ? label(u * 32 + lane) : -1;
#pragma unroll
      for (int f = 0; f < F; ++f) {
        kept[u][f] = logit(v, f);
        best[f] = fmaxf(best[f], kept[u][f]);
      }
    }
  for (int i = KEEP * 32 + lane; i < len; i += 32) {
    const int v = label(i);
#pragma unroll
    for (int f = 0; f < F; ++f) best[f] = fmaxf(best[f], logit(v, f));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
#pragma unroll
    for (int f = 0; f < F; ++f) best[f] = fmaxf(best[f], __shfl_xor_sync(0xffffffffu, best[f], d));
  auto put = [&](int i, int f, float logit) {
    const float x = logit - best[f];
    if (x >= kImpossible) least[f] = fminf(least[f], x);
    em[(int64_t)f * a.pitch + i] = emission_word(x);
  };
#pragma unroll
  for (int f = 0; f < F; ++f)
    if (f < count) {
#pragma unroll
      for (int u = 0; u < KEEP; ++u)
        if (u * 32 + lane < len) put(u * 32 + lane, f, kept[u][f]);
      if (lane == 0) {
        put(a.S + 1, f, logit(a.blank, f));
        em[(int64_t)f * a.pitch + a.S] = 0u;
      }
    }
  for (int i = KEEP * 32 + lane; i < len; i += 32) {
    const int v = label(i);
    for (int f = 0; f < count; ++f) put(i, f, logit(v, f));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
#pragma unroll
    for (int f = 0; f < F; ++f) least[f] = fminf(least[f], __shfl_xor_sync(0xffffffffu, least[f], d));
#pragma unroll
  for (int f = 0; f < F; ++f)
    if (f < count) {
      const bool far = least[f] < kLowest;
      if (far) write_far_emissions<T>(x + f * a.ld_t, em + (int64_t)f * a.pitch, targets, len, a.S, a.blank, a.V, best[f], lane);
      if (lane == f)
        em[(int64_t)f * a.pitch + a.S + 2] = (uint32_t)(int)ceilf(-least[f] * kLog2e) | (far ? kFarSpan : 0u);
    }
}

// what the frame adds to -log Z: its emissions are against `best` instead of the softmax's denominator.  Natural, so that
// a difference of the type's lowest value stays finite.
__device__ __forceinline__ float frame_norm(const Online& o, float best) {
  return logf(o.sum) + (best == -INFINITY ? 0.f : o.top - best);
}

constexpr int kRowThreads = 256;
// Up to it a warp takes a row, beyond it a CTA.  Loss and gradient in a warp | in a CTA, bf16: 48 x 384 x 2048 61 + 47 |
// 89 + 94 us, 48 x 384 x 4096 78 + 88 | 100 + 109, 48 x 128 x 8192 51 + 66 | 51 + 53; but one utterance of 60 frames
// waits for its rows: 22.5 + 10.2 | 20.5 + 8.2 at 2048 classes, 24.6 + 14.3 | 20.5 + 8.2 at 4096.
constexpr int kWarpRowV = 2048;

// Frames of one utterance that a warp takes: two, which share what is looked up of the transcript, where that leaves
// 16 warps an SM; a CTA takes one.  48 x 1536 x 348 with 300 labels: rows and gradient 47 and 59 us, with three frames
// 55 and 71, with four 70 and 75.
int warp_frames(const CtcArgs& a) { return (int64_t)a.B * a.T >= 32 * device_sm_count() ? 2 : 1; }

// block (frames, utterance); the last block of an utterance plans it
template <typename T, int F, bool WARP_ROW>
__global__ void __launch_bounds__(kRowThreads) ctc_rows_kernel(CtcArgs a) {
  const int b = blockIdx.y;
  if (blockIdx.x == gridDim.x - 1) return plan_utterance(a, b);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = WARP_ROW ? (blockIdx.x * (kRowThreads / 32) + warp) * F : blockIdx.x;
  const int count = min(min(__ldg(a.input_lengths + b), a.T) - t, F);
  if (count <= 0) return;
  const T* x = static_cast<const T*>(a.logits) + b * a.ld_b + t * a.ld_t;
  const int64_t frame = (int64_t)b * a.T + t;
  Online o[F];
  if (WARP_ROW) {
#pragma unroll
    for (int f = 0; f < F; ++f)
      if (f < count) o[f] = scan_row<T, 32>(x + f * a.ld_t, a.V, lane);
  } else {
    __shared__ Online part[kRowThreads / 32];
    o[0] = scan_row<T, kRowThreads>(x, a.V, threadIdx.x);
    if (lane == 0) part[warp] = o[0];
    __syncthreads();
    if (warp > 0) return;
    o[0] = part[0];
#pragma unroll
    for (int i = 1; i < kRowThreads / 32; ++i) o[0] = online_join(o[0], part[i]);
  }
  float best[F];
  write_emissions<T, F, WARP_ROW ? 10 : 1>(a, x, frame, count, b, lane, best);
#pragma unroll
  for (int f = 0; f < F; ++f)
    if (lane == f && f < count) {
      a.stats[frame + f] = make_float2(o[f].top, o[f].sum);
      a.norms[frame + f] = frame_norm(o[f], best[f]);
    }
}

// ---- lattice ---------------------------------------------------------------------------------------------------------
// Two CTAs an utterance, a cluster: one walks alpha from the first frame, one beta from the last, the same code on
// reversed frames and labels.  They meet in the middle (frame h): until there each stores its states, behind it each
// reads the other's and multiplies, so the posteriors need no second chain and half of each chain is stored.  Beta
// carries its emission; the posterior takes the other side's sum before its own emission, so none counts twice.
//
// A pair (blank i, label i) is the unit; a lane holds NP pairs, a warp 32 NP.  A step needs the label of the pair
// below: one shuffle within the warp.  Across warps, each keeps the top HL lanes' worth of the warp below it as extra
// pairs of its own at its low end; H steps reach at most 2 H states, so they are refreshed every H frames, and one
// barrier serves H steps.  Emissions and the other side's states come H frames at a time by bulk copies.
//
// Within a block of H frames a lane may hold its states as fp64 against one exponent, the largest of the states that
// can reach it: a step is then two products and three multiply-adds a pair (behind the meeting, which wants the sums
// before the emission: two additions, a multiply-add, two products), and the stored words are used as they are.  A warp takes this form where its states (else the states of each lane's reach) and the block's emissions
// together span no more than kFastSpan octaves, which keeps every state of weight a normal number, and no lane's states
// lie out of the factor's reach from the lane above; any other block, and one that is not whole, runs on the exponent
// of every state, at three times the instructions.
//
// Bound by the instructions of one warp a scheduler: at 48 utterances of 1536 frames with 300 labels (195 us) a step
// takes 171 cycles before the meeting and 357 behind it, 60 of them a block's begin and end; HBM and the fp64 pipe wait.
// Posteriors on warps of their own, a few frames behind the walkers, came to 236-335 us: both want the same scheduler.
constexpr int kFastSpan = 1850;
constexpr int kFastBias = 900;                // the largest state starts a block at 2^900

template <int NP, int H>
__host__ __device__ constexpr int halo_lanes() { return (H + NP - 1) / NP; }

__host__ __device__ constexpr int lattice_warps(int pairs, int NP, int HL) {
  return pairs <= 32 * NP ? 1 : 1 + (pairs - 32 * NP + (32 - HL) * NP - 1) / ((32 - HL) * NP);
}

// Four warps at most hold up to three pairs a lane; one more warp fetches the frames and adds up the blanks.
// WIDE: every block on the exponents of its states, every state stored with its own, and frames of either emission words.
// Otherwise true comes back, on both sides, where the utterance has to be walked so: no posterior is written yet, and the
// loss where only the posteriors ask for it (again = 1), not the emissions (2).  3 stands for a wait that has run out.
// HOLD: the self-test's, which leaves a copy out.
template <int NP, int H, int NBUF, bool GRAD, bool WIDE, bool HOLD>
__device__ __forceinline__ bool lattice_walk(const CtcArgs& a, int nw) {
  constexpr int HL = halo_lanes<NP, H>(), NS = 2 * NP;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[NBUF];
  __shared__ double norms_sum;
  __shared__ float zm[32];
  __shared__ int ze[32];
  const int dir = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int n = __ldg(a.input_lengths + b), len = __ldg(a.target_lengths + b);
  kernel_wait_ahead();
  const bool bad = a.bad[b] || n < 0 || n > a.T;
  if (bad || n == 0) {                             // both CTAs of the cluster leave here
    if (dir == 0 && tid == 0) {
      const float raw = bad ? NAN : len == 0 ? 0.f : INFINITY;
      a.raw_loss[b] = raw;
      a.loss[b] = a.zero_infinity && raw == INFINITY ? 0.f : raw;
    }
    return false;
  }
  const int pitch = a.pitch, spitch = a.state_pitch, brow = nw * 32 + 4;
  const int64_t frame0 = (int64_t)b * a.T;
  // shared memory: emission ring, state ring (GRAD), halo exchange, blanks' partial sums (GRAD)
  uint32_t* em_ring = reinterpret_cast<uint32_t*>(smem);
  uint32_t* st_ring = em_ring + NBUF * H * pitch;
  float2* halo = reinterpret_cast<float2*>(st_ring + (GRAD ? NBUF * H * spitch : 0));   // [2][nw][HL * NS]
  float* blanks = reinterpret_cast<float*>(halo + 2 * nw * HL * NS);                     // [2][H][nw * 32 + 4]

  if (tid == 0) {
    for (int i = 0; i < NBUF; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  const bool producer = w == nw;
  // this lane's pairs: where their labels lie in a frame, whether a jump from the label below is allowed (0) or not
  const int i0 = w * (32 - HL) * NP + lane * NP;
  const bool own = !producer && (w == 0 || lane >= HL);
  const bool active = !producer && i0 - lane * NP <= len;   // a warp beyond the last pair only keeps the barriers
  const int* targets = a.targets + (int64_t)b * a.S;
  const int step = dir ? -1 : 1;
  int slot[NP], pen[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int i = i0 + j;
    const int li = dir ? len - 1 - i : i;
    slot[j] = i < len ? li : a.S;
    pen[j] = kZeroExp;
    if (i >= 1 && i < len) {
      const int later = __ldg(targets + (dir ? li + 1 : li)), earlier = __ldg(targets + (dir ? li : li - 1));
      if (later != a.blank && later != earlier) pen[j] = 0;
    }
  }
  const int blanks_here = own ? min(max(len + 1 - i0, 0), NP) : 0, labels_here = own ? min(max(len - i0, 0), NP) : 0;
  // The other side's order is the reverse: its pair len - i has this pair's blank, its pair len - 1 - i this label.
  // So this lane reads its pairs q0, q0 - 1, ..., q0 - NP; they lie in two of its lanes at most, whose references are
  // found behind the states: pairs q0 - from_lo and below are the lower lane's.
  const int q0 = len - i0;
  auto owner = [&](int q) {
    q = max(q, 0);
    const int ow = q < 32 * NP ? 0 : 1 + (q - 32 * NP) / ((32 - HL) * NP);
    return ow * 32 + (q - ow * (32 - HL) * NP) / NP;
  };
  const int ref_hi = 2 * pitch + owner(q0), ref_lo = 2 * pitch + owner(q0 - NP);
  int from_lo = NP + 1;
#pragma unroll
  for (int j = NP; j >= 1; --j)
    if (owner(q0 - j) != owner(q0)) from_lo = j;

  float m[NS];
  int e[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    m[s] = 1.f;
    e[s] = i0 == 0 && s == 0 && !producer ? 0 : kZeroExp;   // one path, before the first frame
  }
  // the frames' normalisers, by the warp that has the time
  double norm = 0.0;
  if (dir == 0 && producer)
    for (int t = lane; t < n; t += 32) norm += (double)a.norms[frame0 + t];
  __syncthreads();

  const int h = (n + 1) / 2, n1 = dir ? n - h : h;  // this side's frames before the meeting
  int issued = 0, waited = 0, blocks = 0, parity = 0;
  bool fail = false;
  int again = 0;

  // frames [k, k + cnt) of this side's order are rows lo, lo + 1, ...
  auto issue = [&](int k, int cnt, bool states) {
    const int lo = dir ? n - k - cnt : k, buf = issued % NBUF;
    const uint32_t be = cnt * pitch * 4, bs = states ? cnt * spitch * 4 : 0;
    mbar_arrive_expect_tx(&full[buf], be + bs);
    if (!HOLD || b > 0 || k > (states ? n1 : 0) || a.withhold != 1 + dir + 2 * states)
      bulk_load(em_ring + buf * H * pitch, a.post + (frame0 + lo) * pitch, be, &full[buf]);
    if (states) bulk_load(st_ring + buf * H * spitch, a.states + (frame0 + lo) * spitch, bs, &full[buf]);
    ++issued;
  };
  auto refresh_halo = [&]() {
    if (w > 0 && lane < HL) {
      const float2* src = halo + ((parity ^ 1) * nw + w - 1) * HL * NS + lane * NS;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        m[s] = src[s].x;
        e[s] = __float_as_int(src[s].y);
      }
    }
  };
  auto publish_halo = [&]() {
    if (lane >= 32 - HL) {
      float2* dst = halo + (parity * nw + w) * HL * NS + (lane - 32 + HL) * NS;
#pragma unroll
      for (int s = 0; s < NS; ++s) dst[s] = make_float2(m[s], __int_as_float(e[s]));
    }
  };
  float um;
  int ue;                                          // the label of the pair below this lane's
  auto fetch_below = [&]() {
    um = __shfl_up_sync(0xffffffffu, m[NS - 1], 1);
    ue = __shfl_up_sync(0xffffffffu, e[NS - 1], 1);
    if (lane == 0) ue = kZeroExp;
  };
  // sums into every state, without the emission: (pm, pe)
  auto gather = [&](float (&pm)[NS], int (&pe)[NS]) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const float bm = m[2 * j], lm = m[2 * j + 1], vm = j ? m[j ? 2 * j - 1 : 0] : um;
      const int be = e[2 * j], le = e[2 * j + 1], ve = j ? e[j ? 2 * j - 1 : 0] : ue, je = ve + pen[j];
      const int eb = max(be, ve), el = max(max(le, be), je);
      pe[2 * j] = eb;
      pm[2 * j] = fmaf(bm, pow2i(be - eb), vm * pow2i(ve - eb));
      pe[2 * j + 1] = el;
      pm[2 * j + 1] = fmaf(lm, pow2i(le - el), fmaf(bm, pow2i(be - el), vm * pow2i(je - el)));
    }
  };

  float zinv = 0.f;
  int zexp = 0;
  // One block of frames on the exponent of every state; m grows by less than 2^2.6 a frame in between.
  auto frames = [&](auto second, int k, int cnt, const uint32_t* em, const uint32_t* st) {
    constexpr bool SECOND = decltype(second)::value;
    const int first = dir ? cnt - 1 : 0;
    const int64_t frame = frame0 + (dir ? n - 1 - k : k);
    em += first * pitch;
    st += first * spitch;
    [[maybe_unused]] float* post = a.post + frame * pitch;
    [[maybe_unused]] uint32_t* dst = a.states + frame * spitch;
    [[maybe_unused]] uint32_t* upper = a.upper + frame * pitch;
    [[maybe_unused]] float* bl = blanks + parity * H * brow + tid;
    [[maybe_unused]] uint32_t ahead[NP + 1];       // the next frame's upper halves, of pairs q0 - j
    auto load_upper = [&]() {
      if constexpr (SECOND && WIDE)
#pragma unroll
        for (int j = 0; j <= NP; ++j) ahead[j] = __ldcg(upper + max(q0 - j, 0));
    };
    load_upper();
    for (int f = 0; f < cnt; ++f) {
      float pm[NS];
      int pe[NS];
      fetch_below();
      gather(pm, pe);
      if constexpr (WIDE) {
        const bool far = em[a.S + 2] >= kFarSpan;
        const int shift = far ? kFarShift : 20, bias = far ? kFarBias : 1023;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const uint32_t x = em[s & 1 ? slot[s / 2] : a.S + 1], field = x >> shift;
          m[s] = pm[s] * __uint_as_float(((x << (23 - shift)) & 0x7FFFFFu) | 0x3F800000u);
          e[s] = max(pe[s] + (field == 0 ? kZeroExp : (int)field - bias), kZeroExp);
        }
      } else {
        if constexpr (!SECOND)
          if (em[a.S + 2] >= kFarSpan) again = 2;  // this walk's numbers are void from here on
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const uint32_t x = em[s & 1 ? slot[s / 2] : a.S + 1];
          m[s] = pm[s] * word_mantissa(x);
          e[s] = max(pe[s] + (x < kWordOne ? kZeroExp : (int)(x >> 20) - 1023), kZeroExp);
        }
      }
      if constexpr (SECOND && WIDE) {
        uint32_t up[NP + 1];
#pragma unroll
        for (int j = 0; j <= NP; ++j) up[j] = ahead[j];
        upper += step * pitch;
        if (f + 1 < cnt) load_upper();
        auto joint = [&](int j, int s, float pm, int pe) {         // with state s (0 blank, 1 label) of the pair q0 - j
          const uint32_t v = st[2 * max(q0 - j, 0) + s], u = up[j] >> (16 * s) & 0xFFFFu;
          return u == 0 ? 0.f : pm * (wide_mantissa(v) * zinv) * pow2i(wide_exponent(v, u) - zexp + pe);
        };
        float blank = 0.f;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          if (j < blanks_here) blank += joint(j, 0, pm[2 * j], pe[2 * j]);
          if (j < labels_here) post[slot[j]] = joint(j + 1, 1, pm[2 * j + 1], pe[2 * j + 1]);
        }
        bl[f * brow] = blank;
        post += step * pitch;
        st += step * spitch;
      } else if constexpr (SECOND) {
        const int rh = (int)st[ref_hi] - zexp, rl = (int)st[ref_lo] - zexp;
        float blank = 0.f;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const uint32_t vb = st[2 * max(q0 - j, 0)], vl = st[2 * max(q0 - j - 1, 0) + 1];
          const int eb = (int)(vb >> 20) + (j < from_lo ? rh : rl) + pe[2 * j];
          const int el = (int)(vl >> 20) + (j + 1 < from_lo ? rh : rl) + pe[2 * j + 1];
          const float gb = vb < kWordOne ? 0.f : pm[2 * j] * (word_mantissa(vb) * zinv) * pow2i(eb);
          const float gl = vl < kWordOne ? 0.f : pm[2 * j + 1] * (word_mantissa(vl) * zinv) * pow2i(el);
          if (j < blanks_here) blank += gb;
          if (j < labels_here) post[slot[j]] = gl;
        }
        bl[f * brow] = blank;
        post += step * pitch;
        st += step * spitch;
      } else if constexpr (GRAD && WIDE) {
#pragma unroll
        for (int j = 0; j < NP; ++j)
          if (j < blanks_here) {
            uint32_t ub, ul;
            const uint32_t vb = to_wide(m[2 * j], e[2 * j], ub), vl = to_wide(m[2 * j + 1], e[2 * j + 1], ul);
            *reinterpret_cast<uint2*>(dst + 2 * (i0 + j)) = make_uint2(vb, vl);
            upper[i0 + j] = ub | ul << 16;
          }
        dst += step * spitch;
        upper += step * pitch;
      } else if constexpr (GRAD) {
        int ref = e[0];
#pragma unroll
        for (int s = 1; s < NS; ++s) ref = max(ref, e[s]);
#pragma unroll
        for (int s = 0; s < NS; ++s)
          if (own && e[s] >= kZeroBelow && e[s] < ref - kWordSpan) again = max(again, 1);
#pragma unroll
        for (int j = 0; j < NP; ++j)
          if (j < blanks_here)
            *reinterpret_cast<uint2*>(dst + 2 * (i0 + j)) =
                make_uint2(to_word(m[2 * j], e[2 * j] - ref), to_word(m[2 * j + 1], e[2 * j + 1] - ref));
        if (own) dst[2 * pitch + tid] = (uint32_t)(ref - 1023);
        dst += step * spitch;
      }
      em += step * pitch;
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) {                 // leading ones out of m
      const int bits = __float_as_int(m[s]), d = (bits >> 23) - 127;
      m[s] = __int_as_float(bits - (d << 23));
      e[s] += d;
    }
  };

  // Whether a whole block can run as fp64 against E, and E: the largest exponent of the warp's states, or of those that
  // reach this lane.
  int E = 0;
  double below = 0.0;                              // the label below comes against its own lane's E
  auto fast_block = [&](const uint32_t* em) {
    int hi = e[0], lo = INT_MAX;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      hi = max(hi, e[s]);
      lo = min(lo, e[s] < kZeroBelow ? INT_MAX : e[s]);
    }
    const int span = __reduce_add_sync(0xffffffffu, lane < H ? em[lane * pitch + a.S + 2] : 0u);
    const int top = __reduce_max_sync(0xffffffffu, hi), least = __reduce_min_sync(0xffffffffu, lo);
    E = top;
    below = lane == 0 ? 0.0 : 1.0;
    if (least == INT_MAX || top - least + span <= kFastSpan) return true;
#pragma unroll
    for (int d = 1; d <= HL; d *= 2) {
      const int uh = __shfl_up_sync(0xffffffffu, hi, d), ul = __shfl_up_sync(0xffffffffu, lo, d);
      if (lane >= d) {
        hi = max(hi, uh);
        lo = min(lo, ul);
      }
    }
    E = hi;
    // Where nothing but zeros reaches a lane or the one below it, nothing comes from below within the block.  A lane
    // below that lies further down than the factor reaches still counts: its path can be the one that goes on.
    const int under = __shfl_up_sync(0xffffffffu, E, 1), lower = under - E;
    const bool closed = lane == 0 || E < kZeroBelow || under < kZeroBelow, held = lower >= -1000 && lower <= 900;
    below = __hiloint2double(closed || !held ? 0 : (lower + 1023) << 20, 0);
    return __all_sync(0xffffffffu, (lo == INT_MAX || hi - lo + span <= kFastSpan) && (closed || held)) != 0;
  };
  auto fast_frames = [&](auto second, int k, const uint32_t* em, const uint32_t* st) {
    constexpr bool SECOND = decltype(second)::value;
    const int first = dir ? H - 1 : 0;
    const int64_t frame = frame0 + (dir ? n - 1 - k : k);
    em += first * pitch;
    st += first * spitch;
    [[maybe_unused]] float* post = a.post + frame * pitch;
    [[maybe_unused]] uint32_t* dst = a.states + frame * spitch;
    [[maybe_unused]] float* bl = blanks + parity * H * brow + tid;
    double v[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const uint32_t bits = __float_as_uint(m[s]);
      const int d = e[s] - E;
      v[s] = d < -kFastSpan - 50 ? 0.0 : __hiloint2double((int)(bits >> 3) + ((d + 896 + kFastBias) << 20), (int)(bits << 29));
    }
    uint32_t x[NP + 1];
    [[maybe_unused]] uint2 sv[NP + 1];
    [[maybe_unused]] int rh = 0, rl = 0;
    auto load_em = [&]() {
#pragma unroll
      for (int j = 0; j < NP; ++j) x[j] = em[slot[j]];
      x[NP] = em[a.S + 1];
    };
    auto load_st = [&]() {
      if constexpr (SECOND) {
        rh = (int)st[ref_hi];
        rl = (int)st[ref_lo];
#pragma unroll
        for (int j = 0; j <= NP; ++j) sv[j] = *reinterpret_cast<const uint2*>(st + 2 * max(q0 - j, 0));
      }
    };
    load_em();
    load_st();
    double u = __shfl_up_sync(0xffffffffu, v[NS - 1], 1);
    // as far unrolled as the instruction cache holds: three pairs and eight frames of the second half took 2.2 times
    // as long as two
    constexpr int UNROLL = !SECOND ? 8 : NP == 1 ? 4 : 2;
#pragma unroll(UNROLL)
    for (int f = 0; f < H; ++f) {
      double p[NP + 1], pre[NS];
#pragma unroll
      for (int j = 0; j <= NP; ++j) p[j] = __hiloint2double((int)x[j], 0);
      const bool more = f + 1 < H;
      if (more) {
        em += step * pitch;
        load_em();
      }
      const double ub = u * below;
      // from the top pair down: each reads the label below it before that changes
#pragma unroll
      for (int j = NP - 1; j >= 0; --j) {
        const double ul = j ? v[j ? 2 * j - 1 : 0] : ub;
        if constexpr (SECOND) {
          pre[2 * j + 1] = fma(pen[j] == 0 ? 1.0 : 0.0, ul, v[2 * j + 1] + v[2 * j]);
          pre[2 * j] = v[2 * j] + ul;
          v[2 * j + 1] = pre[2 * j + 1] * p[j];
          v[2 * j] = pre[2 * j] * p[NP];
        } else {                                   // the shortest chain: one multiply-add behind the shuffle, two in a lane
          v[2 * j + 1] = fma(pen[j] == 0 ? p[j] : 0.0, ul, fma(p[j], v[2 * j + 1], p[j] * v[2 * j]));
          v[2 * j] = fma(p[NP], ul, p[NP] * v[2 * j]);
        }
        if (j == NP - 1 && more) u = __shfl_up_sync(0xffffffffu, v[NS - 1], 1);
      }
      if constexpr (SECOND) {
        // the other side's value against 2^(zexp - E + kFastBias), as fp64; what lies above its range meets a zero
        const int sh = rh + E - kFastBias - zexp + 1023, sl = rl + E - kFastBias - zexp + 1023;
        auto other = [&](uint32_t word, int shift) {
          const int field = min(max((int)(word >> 20) + shift, 0), 2046);
          return __hiloint2double(word < kWordOne ? 0 : (int)((field << 20) | (word & (kWordOne - 1))), 0);
        };
        float blank = 0.f;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float gb = to_float(pre[2 * j] * other(sv[j].x, j < from_lo ? sh : sl)) * zinv;
          const float gl = to_float(pre[2 * j + 1] * other(sv[j + 1].y, j + 1 < from_lo ? sh : sl)) * zinv;
          if (j < blanks_here) blank += gb;
          if (j < labels_here) post[slot[j]] = gl;
        }
        if (more) {
          st += step * spitch;
          load_st();
        }
        bl[f * brow] = blank;
        post += step * pitch;
      } else if constexpr (GRAD) {
        auto word = [](double d) { return (uint32_t)__double2hiint(d) + ((uint32_t)__double2loint(d) >> 31); };
#pragma unroll
        for (int j = 0; j < NP; ++j)
          if (j < blanks_here) *reinterpret_cast<uint2*>(dst + 2 * (i0 + j)) = make_uint2(word(v[2 * j]), word(v[2 * j + 1]));
        if (own) dst[2 * pitch + tid] = (uint32_t)(E - kFastBias - 1023);
        dst += step * spitch;
      }
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const long long bits = __double_as_longlong(v[s]) + (1ll << 28);   // to_float cuts: rounds to nearest
      const int hi = (int)(bits >> 32);
      const bool zero = hi < (int)kWordOne;
      m[s] = zero ? 1.f : to_float(__hiloint2double((hi & (int)(kWordOne - 1)) | 0x3FF00000, (int)bits));
      e[s] = zero ? kZeroExp : (hi >> 20) - 1023 - kFastBias + E;
    }
  };
  // The fetching warp waits for the frames one block ahead, so the barrier behind a block also hands over the next.
  auto wait_block = [&](int block) {
    const bool ok = mbar_wait_bounded(&full[block % NBUF], (block / NBUF) & 1, nullptr, kStatusTimeoutCtc);
    if (ok) ++waited;
    return ok;
  };
  auto walk = [&](int k0, int k1, auto second) {
    constexpr bool SECOND = decltype(second)::value;
    if (k0 >= k1) return;
    const int vecs = lattice_warps(len + 1, NP, HL) * 8;        // of four blanks a frame
    auto add_blanks = [&](int k, int cnt, int half) {           // 32 / H lanes a frame
      const int f = lane / (32 / H);
      float s = 0.f;
      const float4* src = reinterpret_cast<const float4*>(blanks + (half * H + f) * brow);
      if (f < cnt)
        for (int i = lane % (32 / H); i < vecs; i += 32 / H) {
          const float4 q = src[i];
          s += (q.x + q.y) + (q.z + q.w);
        }
#pragma unroll
      for (int d = 16 / H; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (f < cnt && lane % (32 / H) == 0) a.post[(frame0 + (dir ? n - 1 - k - f : k + f)) * pitch + a.S + 1] = s;
    };
    bool ok = true;
    if (producer) {
      if (lane == 0)
        for (int u = 0; u < NBUF; ++u)
          if (k0 + u * H < k1) issue(k0 + u * H, min(H, k1 - k0 - u * H), SECOND);
      ok = wait_block(blocks);
    }
    fail = __syncthreads_or(!ok);
    for (int k = k0; k < k1 && !fail; k += H) {
      const int cnt = min(H, k1 - k), buf = blocks % NBUF;
      if (producer) {
        const int next = k + (NBUF - 1) * H;                     // into the buffer of the block before this one
        if (lane == 0 && k > k0 && next < k1) issue(next, min(H, k1 - next), SECOND);
        if constexpr (SECOND)
          if (k > k0) add_blanks(k - H, H, parity ^ 1);
        if (k + H < k1) ok = wait_block(blocks + 1);
      } else if (active) {
        refresh_halo();
        const uint32_t* em = em_ring + buf * H * pitch;
        const uint32_t* st = st_ring + buf * H * spitch;
        bool fast = false;
        if constexpr (!WIDE) fast = cnt == H && fast_block(em);
        if (fast) {
          if constexpr (!WIDE) fast_frames(second, k, em, st);
        } else {
          frames(second, k, cnt, em, st);
        }
        publish_halo();
      }
      fail = __syncthreads_or(!ok);
      parity ^= 1;
      ++blocks;
    }
    if constexpr (SECOND)
      if (producer && !fail) {
        const int last = (k1 - k0 - 1) / H * H;
        add_blanks(k0 + last, k1 - k0 - last, parity ^ 1);
      }
  };
  auto drain = [&]() {                             // after a wait that ran out: the copies under way land first
    if (producer && lane == 0)
      for (int i = waited; i < issued; ++i)
        mbar_wait_bounded(&full[i % NBUF], (i / NBUF) & 1, nullptr, kStatusTimeoutCtc);
  };

  if (!producer) publish_halo();
  parity ^= 1;
  __syncthreads();
  walk(0, n1, std::false_type{});

  // the meeting: Z = sum over the states of this side's sum into them times the other side's value
  // (a place of its own for either walk: the other side may still be at the first one's meeting)
  float2* mine = a.exchange + (((int64_t)b * 2 + WIDE) * 2 + dir) * 2 * pitch;
  const float2* theirs = a.exchange + (((int64_t)b * 2 + WIDE) * 2 + (dir ^ 1)) * 2 * pitch;
#pragma unroll
  for (int j = 0; j < NP; ++j)
    if (j < blanks_here) {
      mine[2 * (i0 + j)] = make_float2(m[2 * j], __int_as_float(e[2 * j]));
      mine[2 * (i0 + j) + 1] = make_float2(m[2 * j + 1], __int_as_float(e[2 * j + 1]));
    }
  if (fail) again = 3;
  if (again) atomicMax(a.again + b, again);        // any lane's, either side's
  // the states were stored by plain stores and are fetched by bulk copies of the other CTA
  asm volatile("fence.proxy.async;" ::: "memory");
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  asm volatile("fence.proxy.async;" ::: "memory");
  if (fail) {
    drain();
    return false;
  }
  again = __ldcg(a.again + b);
  {
    int top = 2 * kZeroExp;
    float total = 0.f;
    if (active) {
      float pm[NS];
      int pe[NS];
      refresh_halo();
      fetch_below();
      gather(pm, pe);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const float2 none = make_float2(1.f, __int_as_float(kZeroExp));
        const float2 vb = j < blanks_here ? __ldcg(theirs + 2 * (q0 - j)) : none;
        const float2 vl = j < labels_here ? __ldcg(theirs + 2 * (q0 - j - 1) + 1) : none;
        pm[2 * j] *= vb.x;
        pe[2 * j] += __float_as_int(vb.y);
        pm[2 * j + 1] *= vl.x;
        pe[2 * j + 1] += __float_as_int(vl.y);
      }
#pragma unroll
      for (int s = 0; s < NS; ++s) top = max(top, pe[s]);
      top = __reduce_max_sync(0xffffffffu, top);
#pragma unroll
      for (int s = 0; s < NS; ++s) total = fmaf(pm[s], pow2i(pe[s] - top), total);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    }
    if (producer) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) norm += __shfl_xor_sync(0xffffffffu, norm, d);
      if (lane == 0) norms_sum = norm;
    } else if (lane == 0) {
      zm[w] = total;
      ze[w] = top;
    }
    __syncthreads();
    if (again >= (WIDE ? 3 : 2)) return !WIDE;
    top = ze[0];
    for (int i = 1; i < nw; ++i) top = max(top, ze[i]);
    total = 0.f;
    for (int i = 0; i < nw; ++i) total += zm[i] * pow2i(ze[i] - top);
    const bool exists = top > kZeroBelow;
    if ((!WIDE || again == 2) && dir == 0 && tid == 0) {
      norm = norms_sum;
      float raw = INFINITY;
      if (exists) raw = (float)(norm - ((double)top + log2((double)total)) * 0.6931471805599453);
      if (!(norm > -INFINITY)) raw = NAN;          // a frame of NaN, +inf or nothing but -inf
      a.raw_loss[b] = raw;
      a.loss[b] = a.zero_infinity && raw == INFINITY ? 0.f : raw;
    }
    if (!GRAD || !exists) return false;
    if (!WIDE && again) return true;
    const int bits = __float_as_int(total), k = (bits >> 23) - 127;
    zinv = 1.f / __int_as_float(bits - (k << 23));
    zexp = top + k;
  }
  if constexpr (GRAD) {
    walk(n1, n, std::true_type{});
    if (fail) {                                    // the gradient kernel makes NaN of the posteriors that are not there
      uint32_t here;                               // b: kept to this place in a register, it cost the walk 30 us of 306
      asm volatile("mov.u32 %0, %%ctaid.y;" : "=r"(here));
      a.again[here] = 3;
      drain();
    }
  }
  return false;
}

// A function of its own: its code beside the other walk's took a fifth of that one's speed.  48 utterances of 799 frames
// with 300 labels, all of them walked again: 530 us with the gradient, 178 where none is.
template <int NP, int H, int NBUF, bool GRAD, bool HOLD>
__device__ __noinline__ void lattice_wide(const CtcArgs& a, int nw) {
  if (__ldcg(a.again + blockIdx.y) == 3) return;   // the other side has given up
  __syncthreads();                                 // the first walk's shared memory is free
  lattice_walk<NP, H, NBUF, GRAD, true, HOLD>(a, nw);
}

template <int NP, int H, int NBUF, bool GRAD, bool HOLD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NP < 4 ? 160 : H == 8 ? 288 : 576)
    ctc_lattice_kernel(const __grid_constant__ CtcArgs a, int nw) {
  if (lattice_walk<NP, H, NBUF, GRAD, false, HOLD>(a, nw)) lattice_wide<NP, H, NBUF, GRAD, HOLD>(a, nw);
}

// ---- gradient --------------------------------------------------------------------------------------------------------
// What a frame's gradient is made of: d p = scale * 2^((logit - top) / ln 2).
struct FrameGrad {
  float top, scale, d;
  __device__ __forceinline__ float operator()(float x) const { return scale * ex2_approx((x - top) * kLog2e); }
};

__device__ __forceinline__ FrameGrad frame_grad(const CtcArgs& a, int64_t frame, int b) {
  const float2 st = a.stats[frame];
  const float d = __ldg(a.dloss + b);
  return FrameGrad{st.x, d / st.y, d};
}

// d p over all classes of a frame
template <typename T, int THREADS>
__device__ __forceinline__ void grad_row(const FrameGrad& p, const T* __restrict__ x, T* __restrict__ g, int V, int tid) {
  int head = head_of(g, V), vecs = (V - head) / 8;
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15) != 0) {
    head = V;                                      // another alignment than the gradient's: element by element
    vecs = 0;
  }
  for (int v = tid; v < head; v += THREADS) g[v] = from_f32<T>(p(to_f32(x[v])));
  for (int i = tid; i < vecs; i += THREADS) {
    rows_impl::Vec8<T> r;
#pragma unroll
    for (int q = 0; q < rows_impl::Vec8<T>::Q; ++q)
      r.q[q] = __ldg(reinterpret_cast<const uint4*>(x + head + (int64_t)i * 8) + q);
    float e[8];
    rows_impl::unpack(r, e);
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = p(e[k]);
    rows_impl::pack(e, r);
#pragma unroll
    for (int q = 0; q < rows_impl::Vec8<T>::Q; ++q)
      *(reinterpret_cast<uint4*>(g + head + (int64_t)i * 8) + q) = r.q[q];
  }
  for (int v = head + vecs * 8 + tid; v < V; v += THREADS) g[v] = from_f32<T>(p(to_f32(x[v])));
}

// d (p - posterior) over the transcript's classes of `count` frames that follow one another: the posteriors in the
// order of their classes, a running sum within each class, its last place writes.  One warp; the order is looked up
// once for all frames.
template <typename T, int F>
__device__ __forceinline__ void grad_labels(const CtcArgs& a, const FrameGrad (&p)[F], const T* __restrict__ x,
                                            T* __restrict__ g, int64_t frame, int count, int b, int lane) {
  const float* post = a.post + frame * a.pitch;
  const int2* order = a.order + (int64_t)b * a.pitch;
  const int places = __ldg(a.target_lengths + b) + 1;
  const int2 none = make_int2(-1, -2);
  float carry[F] = {};
  int carry_v = -1;
  int2 here = lane < places ? __ldg(order + lane) : none;
  for (int q0 = 0; q0 < places; q0 += 32) {
    const int q = q0 + lane;
    const int2 ahead = q + 32 < places ? __ldg(order + q + 32) : none;
    const int v = here.y;
    int next = __shfl_down_sync(0xffffffffu, v, 1);
    const int first_ahead = __shfl_sync(0xffffffffu, ahead.y, 0);
    if (lane == 31) next = first_ahead;
    const bool last = here.x >= 0 && next != v;
    float joins[6];                                // 1 where the value that far below is of the same class
    joins[5] = v == carry_v ? 1.f : 0.f;
#pragma unroll
    for (int k = 0; k < 5; ++k) {                  // sorted: equal 2^k below means one class in between
      const int uv = __shfl_up_sync(0xffffffffu, v, 1 << k);
      joins[k] = lane >= (1 << k) && uv == v ? 1.f : 0.f;
    }
#pragma unroll
    for (int f = 0; f < F; ++f) {
      if (f >= count) break;
      float s = here.x < 0 ? 0.f : post[(int64_t)f * a.pitch + here.x];
#pragma unroll
      for (int k = 0; k < 5; ++k) s = fmaf(joins[k], __shfl_up_sync(0xffffffffu, s, 1 << k), s);
      s = fmaf(joins[5], carry[f], s);
      if (last) g[(int64_t)f * a.V + v] = from_f32<T>(p[f](to_f32(x[f * a.ld_t + v])) - p[f].d * s);
      carry[f] = __shfl_sync(0xffffffffu, s, 31);
    }
    carry_v = __shfl_sync(0xffffffffu, v, 31);
    here = ahead;
  }
}

template <typename T, int THREADS>
__device__ __forceinline__ void fill_row(T* __restrict__ g, int V, float value, int tid) {
  const int head = head_of(g, V), vecs = (V - head) / 8;
  if (tid < head) g[tid] = from_f32<T>(value);
  const float f[8] = {value, value, value, value, value, value, value, value};
  rows_impl::Vec8<T> r;
  rows_impl::pack(f, r);
  for (int i = tid; i < vecs; i += THREADS)
#pragma unroll
    for (int q = 0; q < rows_impl::Vec8<T>::Q; ++q)
      *(reinterpret_cast<uint4*>(g + head + (int64_t)i * 8) + q) = r.q[q];
  for (int v = head + vecs * 8 + tid; v < V; v += THREADS) g[v] = from_f32<T>(value);
}

constexpr int kCtaThreads = 512;                 // of a row that a CTA takes (256: 186 us, 512: 178, 1024: 182 at 8 x 384 x 100352 bf16)

template <typename T, int F, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? kRowThreads : kCtaThreads) ctc_grad_kernel(CtcArgs a) {
  constexpr int THREADS = WARP_ROW ? 32 : kCtaThreads;
  const int b = blockIdx.y;
  const int t = WARP_ROW ? (blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5)) * F : blockIdx.x;
  if (t >= a.T) return;
  const int tid = WARP_ROW ? threadIdx.x & 31 : threadIdx.x;
  const int64_t frame = (int64_t)b * a.T + t;
  const T* x = static_cast<const T*>(a.logits) + b * a.ld_b + t * a.ld_t;
  T* g = static_cast<T*>(a.dlogits) + frame * a.V;
  const int n = __ldg(a.input_lengths + b);
  const float raw = __ldg(a.raw_loss + b);
  // frames of the utterance: a gradient where there is a finite loss and the lattice came to its end, else zeros or NaN;
  // behind it zeros.  A length out of range makes all its frames NaN.
  const bool fits = n >= 0 && n <= a.T, finite = fabsf(raw) < INFINITY && __ldg(a.again + b) != 3;
  const float other = raw == INFINITY && a.zero_infinity ? 0.f : NAN;
  const int count = fits ? min(n - t, F) : F;      // frames of the F that are not padding
  FrameGrad p[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    if (t + f >= a.T) break;
    if (f < count && finite) {
      p[f] = frame_grad(a, frame + f, b);
      grad_row<T, THREADS>(p[f], x + f * a.ld_t, g + (int64_t)f * a.V, a.V, tid);
    } else {
      fill_row<T, THREADS>(g + (int64_t)f * a.V, a.V, f < count ? other : 0.f, tid);
    }
  }
  if (!finite || count <= 0) return;
  if (WARP_ROW)
    __syncwarp();
  else
    __syncthreads();
  if (tid < 32) grad_labels<T, F>(a, p, x, g, frame, count, b, tid);
}

constexpr size_t kMostSmem = 227 * 1024 - 1024;  // a CTA's, less the static part (of both walks)

template <int NP, int H, int NBUF, bool GRAD, bool HOLD = false>
int launch_lattice(const CtcArgs& a, int nw, cudaStream_t stream) {
  constexpr int HL = halo_lanes<NP, H>(), NS = 2 * NP;
  const size_t smem = (size_t)NBUF * H * a.pitch * 4 + (GRAD ? (size_t)NBUF * H * a.state_pitch * 4 : 0) +
                      (size_t)2 * nw * HL * NS * sizeof(float2) + (GRAD ? (size_t)2 * H * (nw * 32 + 4) * 4 : 0);
  auto* kernel = ctc_lattice_kernel<NP, H, NBUF, GRAD, HOLD>;
  static std::atomic<uint64_t> allowed{0};
  if (int rc = allow_smem((const void*)kernel, kMostSmem, allowed)) return rc;
  return launch_behind(kernel, dim3(2, a.B), (nw + 1) * 32, smem, stream, a, nw);
}

// Pairs a lane: as few as four warps hold (one a scheduler of the SM, so that a step issues in the least time), then
// four pairs and more warps.  Frames a block: 16 where they fit (48 utterances of 1536 frames with 300 labels: 195 us,
// with 8 frames 252 us: about 500 cycles go into a block's begin and end), fewer where the rows get long: beyond 967
// labels two buffers of eight frames, their states and nine warps' blanks come near a CTA's shared memory and at 1000
// past it.  48 utterances, a frame with its gradient: 0.74 us at 967 labels, 0.93 at 968.
struct LatticeShape {
  int NP, H, nw;
};
LatticeShape lattice_shape(int pairs) {
  if (const int nw = lattice_warps(pairs, 1, halo_lanes<1, 16>()); nw <= 4) return {1, 16, nw};
  if (const int nw = lattice_warps(pairs, 2, halo_lanes<2, 16>()); nw <= 4) return {2, 16, nw};
  if (const int nw = lattice_warps(pairs, 3, halo_lanes<3, 16>()); nw <= 4) return {3, 16, nw};
  if (const int nw = lattice_warps(pairs, 4, halo_lanes<4, 8>()); nw <= 8) return {4, 8, nw};
  return {4, 4, lattice_warps(pairs, 4, halo_lanes<4, 4>())};
}

template <bool GRAD>
int launch_lattice_for(const CtcArgs& a, cudaStream_t stream) {
  const LatticeShape s = lattice_shape(a.S + 1);
  if constexpr (GRAD)
    if (a.withhold) return launch_lattice<1, 16, 2, true, true>(a, s.nw, stream);
  if (s.NP == 1) return launch_lattice<1, 16, 2, GRAD>(a, s.nw, stream);
  if (s.NP == 2) return launch_lattice<2, 16, 2, GRAD>(a, s.nw, stream);
  if (s.NP == 3) return launch_lattice<3, 16, 2, GRAD>(a, s.nw, stream);
  if (s.H == 8) return launch_lattice<4, 8, 2, GRAD>(a, s.nw, stream);
  return launch_lattice<4, 4, 2, GRAD>(a, s.nw, stream);
}

// utterances [b0, b0 + 65535): a grid's second extent
CtcArgs batch_part(const CtcArgs& a, int b0, int size) {
  CtcArgs c = a;
  c.B = a.B - b0 < 65535 ? a.B - b0 : 65535;
  const int64_t frames = (int64_t)b0 * a.T;
  c.logits = static_cast<const char*>(a.logits) + b0 * a.ld_b * size;
  c.targets += (int64_t)b0 * a.S;
  c.input_lengths += b0;
  c.target_lengths += b0;
  c.stats += frames;
  c.post += frames * a.pitch;
  c.order += (int64_t)b0 * a.pitch;
  c.raw_loss += b0;
  if (c.loss) c.loss += b0;
  if (c.bad) c.bad += b0;
  if (c.norms) c.norms += frames;
  if (c.again) c.again += b0;
  if (c.exchange) c.exchange += (int64_t)b0 * 8 * a.pitch;
  if (c.states) c.states += frames * a.state_pitch;
  if (c.upper) c.upper += frames * a.pitch;
  if (c.dloss) c.dloss += b0;
  if (c.dlogits) c.dlogits = static_cast<char*>(a.dlogits) + frames * a.V * size;
  return c;
}

template <typename T>
int launch_loss(const CtcArgs& a, cudaStream_t stream) {
  for (int b0 = 0; b0 < a.B; b0 += 65535) {
    const CtcArgs c = batch_part(a, b0, sizeof(T));
    const int frames = warp_frames(a), per = kRowThreads / 32 * frames;
    const dim3 warp_grid((a.T + per - 1) / per + 1, c.B);
    if (a.V > kWarpRowV)
      ctc_rows_kernel<T, 1, false><<<dim3(a.T + 1, c.B), kRowThreads, 0, stream>>>(c);
    else if (frames == 2)
      ctc_rows_kernel<T, 2, true><<<warp_grid, kRowThreads, 0, stream>>>(c);
    else
      ctc_rows_kernel<T, 1, true><<<warp_grid, kRowThreads, 0, stream>>>(c);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
    if (int rc = c.states ? launch_lattice_for<true>(c, stream) : launch_lattice_for<false>(c, stream)) return rc;
  }
  return 0;
}

template <typename T>
int launch_grad(const CtcArgs& a, cudaStream_t stream) {
  for (int b0 = 0; b0 < a.B; b0 += 65535) {
    const CtcArgs c = batch_part(a, b0, sizeof(T));
    const int frames = warp_frames(a), per = kRowThreads / 32 * frames;
    const dim3 warp_grid((a.T + per - 1) / per, c.B);
    if (a.V > kWarpRowV)
      ctc_grad_kernel<T, 1, false><<<dim3(a.T, c.B), kCtaThreads, 0, stream>>>(c);
    else if (frames == 2)
      ctc_grad_kernel<T, 2, true><<<warp_grid, kRowThreads, 0, stream>>>(c);
    else
      ctc_grad_kernel<T, 1, true><<<warp_grid, kRowThreads, 0, stream>>>(c);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
  }
  return 0;
}

}  // namespace ctc_loss_impl

int ctc_pitch(int S) { return (S + 3 + 3) / 4 * 4; }

int ctc_state_pitch(int S) {
  using namespace ctc_loss_impl;
  // the states of the pairs, and a reference for every lane of the warps that hold them
  return 2 * ctc_pitch(S) + 32 * lattice_shape(S + 1).nw;
}

int launch_ctc_loss(const CtcArgs& args, int dtype, cudaStream_t stream) {
  using namespace ctc_loss_impl;
  switch (dtype) {
    case 0: return launch_loss<__nv_bfloat16>(args, stream);
    case 1: return launch_loss<__half>(args, stream);
    default: return launch_loss<float>(args, stream);
  }
}

int launch_ctc_grad(const CtcArgs& args, int dtype, cudaStream_t stream) {
  using namespace ctc_loss_impl;
  switch (dtype) {
    case 0: return launch_grad<__nv_bfloat16>(args, stream);
    case 1: return launch_grad<__half>(args, stream);
    default: return launch_grad<float>(args, stream);
  }
}

}  // namespace gsn
