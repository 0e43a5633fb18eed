// Connectionist temporal classification loss (Graves, Fernandez, Gomez, Schmidhuber, ICML 2006) of the encoder's CTC
// heads, and its gradient with respect to the logits.
//
//   p_t = softmax(logits[t]);  l' = blank l1 blank l2 ... blank, 2 S + 1 states
//   alpha_t(s) = p_t(l'_s) (alpha_{t-1}(s) + alpha_{t-1}(s-1) + [l'_s != blank, l'_s != l'_{s-2}] alpha_{t-1}(s-2))
//   Z = alpha_{n-1}(2S) + alpha_{n-1}(2S-1), loss = -log Z, beta the same from the end (without the emission at t)
//   dlogits[t, v] = dloss (p_t(v) - sum over s with l'_s = v of alpha_t(s) beta_t(s) / Z), 0 for t >= n
//
// Three launches: rows (maximum and sum of exponentials of every frame, the emissions of blank and labels), lattice
// (both chains, the posteriors), gradient.  The emissions are taken against the frame's largest logit, so the frame's
// normaliser stays out of the chain: it cancels in the posteriors, and the loss adds the normalisers in 64 bits.
#include "gsn_kernels.cuh"
#include "gsn_ptx.cuh"

namespace gsn {

namespace ctc_impl {

using rows_impl::from_f32;
using rows_impl::to_f32;

// ---- numbers of the lattice ------------------------------------------------------------------------------------------
// m * 2^e with 1 <= m < 2, or zero: sums over paths leave fp32's range within a few dozen frames, and states thousands
// of octaves below the frame's largest can still carry the whole posterior (a wrong transcript), so every state has
// its own exponent.  A product or sum costs a rounding of the 24-bit m only, wherever the logarithm lies; the
// logarithm itself in fp32 would lose 2^-12 at -4000.
struct Ext {
  float m;
  int e;
};
constexpr int kZeroExp = -(1 << 30);
constexpr float kLowest = -15000.f;   // logits further below the frame's largest count as impossible: the exponents of
                                      // kMaxCtcFrames frames stay within an int

__device__ __forceinline__ Ext ext_zero() { return Ext{0.f, kZeroExp}; }

// 2^d for d <= 0 (0 below the normal range)
__device__ __forceinline__ float pow2_nonpos(int d) { return __int_as_float((max(d, -127) + 127) << 23); }

__device__ __forceinline__ Ext ext_norm(float m, int e) {
  if (m <= 0.f) return ext_zero();
  const int bits = __float_as_int(m);
  const int k = (bits >> 23) - 127;
  return Ext{__int_as_float(bits - (k << 23)), e + k};
}

__device__ __forceinline__ Ext ext_add3(Ext a, Ext b, Ext c) {
  const int e = max(a.e, max(b.e, c.e));
  return ext_norm(fmaf(a.m, pow2_nonpos(a.e - e), fmaf(b.m, pow2_nonpos(b.e - e), c.m * pow2_nonpos(c.e - e))), e);
}

__device__ __forceinline__ Ext ext_mul(Ext a, Ext b) {
  return a.m == 0.f || b.m == 0.f ? ext_zero() : ext_norm(a.m * b.m, a.e + b.e);
}

// exp(a) for a <= 0: 2^k * 2^f with k the nearest integer to a / ln 2
__device__ __forceinline__ Ext ext_exp(float a) {
  if (!(a >= kLowest)) return ext_zero();
  constexpr double kLog2e = 1.4426950408889634;
  constexpr float hi = (float)kLog2e, lo = (float)(kLog2e - (double)hi);
  const float k = rintf(a * hi);
  // the fraction a / ln 2 - k from 1 / ln 2 in two parts: one rounding near zero instead of one near |a|
  const float f = fmaf(a, lo, fmaf(a, hi, -k));
  return ext_norm(exp2f(f), (int)k);
}

// ---- rows ------------------------------------------------------------------------------------------------------------
constexpr int kRowThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kRowThreads) ctc_rows_kernel(CtcArgs a) {
  const int t = blockIdx.x, b = blockIdx.y;
  const int n = __ldg(a.input_lengths + b);
  if (t >= n) return;
  __shared__ float red[2][kRowThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* x = static_cast<const T*>(a.logits) + b * a.ld_b + t * a.ld_t;
  float top = -INFINITY;
  for (int v = threadIdx.x; v < a.V; v += kRowThreads) top = fmaxf(top, to_f32(x[v]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) red[0][warp] = top;
  __syncthreads();
  top = red[0][0];
#pragma unroll
  for (int i = 1; i < kRowThreads / 32; ++i) top = fmaxf(top, red[0][i]);
  float s = 0.f;
  for (int v = threadIdx.x; v < a.V; v += kRowThreads) s += __expf(to_f32(x[v]) - top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) red[1][warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < kRowThreads / 32; ++i) s += red[1][i];
    a.stats[(int64_t)b * a.T + t] = make_float2(top, logf(s));
  }
  float* post = a.post + ((int64_t)b * a.T + t) * (a.S + 1);
  const int len = min(max(__ldg(a.target_lengths + b), 0), a.S);
  for (int i = threadIdx.x; i <= len; i += kRowThreads) {
    const int v = i == 0 ? a.blank : __ldg(a.targets + (int64_t)b * a.S + i - 1);
    post[i] = v >= 0 && v < a.V ? to_f32(x[v]) - top : NAN;   // NaN: a label outside the vocabulary
  }
}

// ---- lattice ---------------------------------------------------------------------------------------------------------
constexpr int kLatticeThreads = 512;

__device__ __forceinline__ int state_label(const CtcArgs& a, const int* targets, int s) {
  return s & 1 ? __ldg(targets + (s >> 1)) : a.blank;
}

__global__ void __launch_bounds__(kLatticeThreads) ctc_lattice_kernel(CtcArgs a) {
  extern __shared__ Ext states[];                  // [2][2 S + 1]
  __shared__ double sums[kLatticeThreads / 32];
  __shared__ float blanks[kLatticeThreads / 32];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int n = __ldg(a.input_lengths + b), len = __ldg(a.target_lengths + b);
  if (n < 0 || n > a.T || len < 0 || len > a.S) {
    if (tid == 0) a.raw_loss[b] = a.loss[b] = NAN;
    return;
  }
  if (n == 0) {
    if (tid == 0) {
      a.raw_loss[b] = len == 0 ? 0.f : INFINITY;
      a.loss[b] = len == 0 || a.zero_infinity ? 0.f : INFINITY;
    }
    return;
  }
  const int* targets = a.targets + (int64_t)b * a.S;
  const int L = 2 * len + 1, full = 2 * a.S + 1;
  float* post = a.post + (int64_t)b * a.T * (a.S + 1);
  float2* alpha = a.alpha ? a.alpha + (int64_t)b * a.T * full : nullptr;
  bool bad = false;
  double norm = 0.0;
  for (int t = tid; t < n; t += kLatticeThreads) norm += (double)__ldg(&a.stats[(int64_t)b * a.T + t].y);
  for (int t = 0; t < n; ++t) {
    Ext* now = states + (t & 1) * L;
    const Ext* old = states + ((t & 1) ^ 1) * L;
    for (int s = tid; s < L; s += kLatticeThreads) {
      const float em = post[(int64_t)t * (a.S + 1) + (s & 1 ? 1 + (s >> 1) : 0)];
      bad |= em != em;
      Ext v;
      if (t == 0) {
        v = s <= 1 ? Ext{1.f, 0} : ext_zero();
      } else {
        const bool skip = (s & 1) && s >= 3 && __ldg(targets + (s >> 1)) != a.blank &&
                          __ldg(targets + (s >> 1)) != __ldg(targets + (s >> 1) - 1);
        v = ext_add3(old[s], s >= 1 ? old[s - 1] : ext_zero(), skip ? old[s - 2] : ext_zero());
      }
      v = ext_mul(v, ext_exp(em));
      now[s] = v;
      if (alpha) alpha[(int64_t)t * full + s] = make_float2(v.m, __int_as_float(v.e));
    }
    __syncthreads();
  }
  const Ext* last = states + ((n - 1) & 1) * L;
  const Ext z = ext_add3(last[L - 1], L >= 2 ? last[L - 2] : ext_zero(), ext_zero());
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) norm += __shfl_xor_sync(0xffffffffu, norm, o);
  if ((tid & 31) == 0) sums[tid >> 5] = norm;
  __syncthreads();
  if (tid == 0) {
    norm = 0.0;
    for (int i = 0; i < kLatticeThreads / 32; ++i) norm += sums[i];
    float loss = INFINITY;
    if (z.m > 0.f) loss = (float)(norm - ((double)z.e + log2((double)z.m)) * 0.6931471805599453);
    if (bad || norm != norm) loss = NAN;
    a.raw_loss[b] = loss;
    a.loss[b] = a.zero_infinity && loss == INFINITY ? 0.f : loss;
  }
  if (!alpha || z.m == 0.f || bad) return;
  // beta, without the emission at t; states hold beta times that emission
  __syncthreads();
  for (int t = n - 1; t >= 0; --t) {
    Ext* now = states + (t & 1) * L;
    const Ext* old = states + ((t & 1) ^ 1) * L;
    float blank = 0.f;
    for (int s = tid; s < L; s += kLatticeThreads) {
      Ext v;
      if (t == n - 1) {
        v = s >= L - 2 ? Ext{1.f, 0} : ext_zero();
      } else {
        const bool skip = (s & 1) && s + 2 < L && __ldg(targets + (s >> 1) + 1) != a.blank &&
                          __ldg(targets + (s >> 1)) != __ldg(targets + (s >> 1) + 1);
        v = ext_add3(old[s], s + 1 < L ? old[s + 1] : ext_zero(), skip ? old[s + 2] : ext_zero());
      }
      const int slot = s & 1 ? 1 + (s >> 1) : 0;
      float* p = post + (int64_t)t * (a.S + 1) + slot;
      now[s] = ext_mul(v, ext_exp(*p));
      const float2 al = alpha[(int64_t)t * full + s];
      const int e = __float_as_int(al.y) + v.e - z.e;
      float gamma = 0.f;
      if (al.x != 0.f && v.m != 0.f) gamma = al.x * v.m / z.m * pow2_nonpos(min(e, 0)) * (e > 0 ? exp2f((float)e) : 1.f);
      if (slot)
        *p = gamma;
      else
        blank += gamma;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) blank += __shfl_xor_sync(0xffffffffu, blank, o);
    if ((tid & 31) == 0) blanks[tid >> 5] = blank;
    __syncthreads();
    if (tid == 0) {
      blank = 0.f;
      for (int i = 0; i < kLatticeThreads / 32; ++i) blank += blanks[i];
      post[(int64_t)t * (a.S + 1)] = blank;
    }
    __syncthreads();
  }
}

// ---- gradient --------------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kRowThreads) ctc_grad_kernel(CtcArgs a) {
  const int t = blockIdx.x, b = blockIdx.y;
  T* g = static_cast<T*>(a.dlogits) + ((int64_t)b * a.T + t) * a.V;
  const int n = __ldg(a.input_lengths + b), len = __ldg(a.target_lengths + b);
  const float raw = __ldg(a.raw_loss + b);
  const bool nan = raw != raw || (raw == INFINITY && !a.zero_infinity);
  const bool padding = t >= n && n >= 0 && n <= a.T;
  if (padding || nan || raw == INFINITY) {
    const float f = !padding && nan ? NAN : 0.f;
    for (int v = threadIdx.x; v < a.V; v += kRowThreads) g[v] = from_f32<T>(f);
    return;
  }
  const T* x = static_cast<const T*>(a.logits) + b * a.ld_b + t * a.ld_t;
  const float2 st = a.stats[(int64_t)b * a.T + t];
  const float d = __ldg(a.dloss + b);
  for (int v = threadIdx.x; v < a.V; v += kRowThreads)
    g[v] = from_f32<T>(d * __expf(to_f32(x[v]) - st.x - st.y));
  __syncthreads();
  // the labels' posteriors, each label by the thread of its first place in the transcript
  const float* post = a.post + ((int64_t)b * a.T + t) * (a.S + 1);
  const int* targets = a.targets + (int64_t)b * a.S;
  for (int i = threadIdx.x; i <= len; i += kRowThreads) {
    const int v = i == 0 ? a.blank : __ldg(targets + i - 1);
    float s = post[i];
    bool first = i == 0 || v != a.blank;
    for (int j = 1; j < i && first; ++j) first = __ldg(targets + j - 1) != v;
    if (!first) continue;
    for (int j = i + 1; j <= len; ++j)
      if (__ldg(targets + j - 1) == v) s += post[j];
    g[v] = from_f32<T>(d * (__expf(to_f32(x[v]) - st.x - st.y) - s));
  }
}

template <typename T>
int launch_loss(const CtcArgs& a, cudaStream_t stream) {
  for (int b0 = 0; b0 < a.B; b0 += 65535) {
    CtcArgs c = a;
    c.B = a.B - b0 < 65535 ? a.B - b0 : 65535;
    const int64_t frames = (int64_t)b0 * a.T;
    c.logits = static_cast<const T*>(a.logits) + b0 * a.ld_b;
    c.targets += (int64_t)b0 * a.S;
    c.input_lengths += b0;
    c.target_lengths += b0;
    c.stats += frames;
    c.post += frames * (a.S + 1);
    c.raw_loss += b0;
    c.loss += b0;
    if (c.alpha) c.alpha += frames * (2 * a.S + 1);
    if (a.T > 0) ctc_rows_kernel<T><<<dim3(a.T, c.B), kRowThreads, 0, stream>>>(c);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
    const size_t smem = (size_t)2 * (2 * a.S + 1) * sizeof(Ext);
    if (smem > 48 * 1024)
      if (cudaError_t e = cudaFuncSetAttribute(ctc_lattice_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem))
        return (int)e;
    ctc_lattice_kernel<<<c.B, kLatticeThreads, smem, stream>>>(c);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
  }
  return 0;
}

template <typename T>
int launch_grad(const CtcArgs& a, cudaStream_t stream) {
  for (int b0 = 0; b0 < a.B; b0 += 65535) {
    CtcArgs c = a;
    c.B = a.B - b0 < 65535 ? a.B - b0 : 65535;
    const int64_t frames = (int64_t)b0 * a.T;
    c.logits = static_cast<const T*>(a.logits) + b0 * a.ld_b;
    c.targets += (int64_t)b0 * a.S;
    c.input_lengths += b0;
    c.target_lengths += b0;
    c.stats += frames;
    c.post += frames * (a.S + 1);
    c.raw_loss += b0;
    c.dloss += b0;
    c.dlogits = static_cast<T*>(a.dlogits) + frames * a.V;
    ctc_grad_kernel<T><<<dim3(a.T, c.B), kRowThreads, 0, stream>>>(c);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
  }
  return 0;
}

}  // namespace ctc_impl

int launch_ctc_loss(const CtcArgs& args, int dtype, cudaStream_t stream) {
  using namespace ctc_impl;
  switch (dtype) {
    case 0: return launch_loss<__nv_bfloat16>(args, stream);
    case 1: return launch_loss<__half>(args, stream);
    default: return launch_loss<float>(args, stream);
  }
}

int launch_ctc_grad(const CtcArgs& args, int dtype, cudaStream_t stream) {
  using namespace ctc_impl;
  switch (dtype) {
    case 0: return launch_grad<__nv_bfloat16>(args, stream);
    case 1: return launch_grad<__half>(args, stream);
    default: return launch_grad<float>(args, stream);
  }
}

}  // namespace gsn
