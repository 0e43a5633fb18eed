// Row operators of fine-tuning: LayerNorm forward and backward, dropout with a residual, and the residual step fused
// with the LayerNorm behind it (the tail of a Conformer block, models/granite_speech_nar/conformer.py:208-209, with
// the dropout that training puts on the feed-forward output).
//
//   m = sum x / D, v = sum (x - m)^2 / D, r = 1 / sqrt(v + eps), xh = (x - m) r
//   forward   y = xh w + b
//   backward  g = dy w, dx = r (g - sum g / D - xh sum(g xh) / D), dw = sum over rows of dy xh, db = sum of dy
//   dropout   h = residual + (u >= threshold ? factor * x : 0), the gradient the same with dout in x's place
//
// Every one of them moves each tensor once, so HBM bounds it.  Tensors are bf16, fp16 or fp32, all arithmetic is fp32.
// Rows are M = B * T frames; with lengths, the frames t >= lengths[b] are padding: their x and dy are not read.
#include "gsn_kernels.cuh"
#include "gsn_ptx.cuh"

#include <cuda_fp16.h>

namespace gsn {

namespace rows_impl {

// ---- eight consecutive elements of a row: the unit of a lane's work and of the dropout generator --------------------
template <typename T>
struct Vec8 {
  static constexpr int Q = sizeof(T) * 8 / 16;   // 16-byte words
  uint4 q[Q];
};

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

__device__ __forceinline__ void unpack(const Vec8<__nv_bfloat16>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = bf16lo_to_f32(w[k]);
    f[2 * k + 1] = bf16hi_to_f32(w[k]);
  }
}
__device__ __forceinline__ void unpack(const Vec8<__half>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    f[2 * k] = p.x;
    f[2 * k + 1] = p.y;
  }
}
__device__ __forceinline__ void unpack(const Vec8<float>& r, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    f[4 * k] = __uint_as_float(r.q[k].x);
    f[4 * k + 1] = __uint_as_float(r.q[k].y);
    f[4 * k + 2] = __uint_as_float(r.q[k].z);
    f[4 * k + 3] = __uint_as_float(r.q[k].w);
  }
}
__device__ __forceinline__ void pack(const float (&f)[8], Vec8<__nv_bfloat16>& r) {
  r.q[0] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void pack(const float (&f)[8], Vec8<__half>& r) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __half2 h = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
    w[k] = *reinterpret_cast<const uint32_t*>(&h);
  }
  r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack(const float (&f)[8], Vec8<float>& r) {
#pragma unroll
  for (int k = 0; k < 2; ++k)
    r.q[k] = make_uint4(__float_as_uint(f[4 * k]), __float_as_uint(f[4 * k + 1]), __float_as_uint(f[4 * k + 2]),
                        __float_as_uint(f[4 * k + 3]));
}

// Columns [col, col + 8) of a row of D elements; columns past D read as zero.  VEC: D % 8 == 0 and 16-byte rows.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, int col, int D, Vec8<T>& r) {
  if (VEC) {
#pragma unroll
    for (int i = 0; i < Vec8<T>::Q; ++i)
      r.q[i] = col < D ? __ldg(reinterpret_cast<const uint4*>(row + col) + i) : make_uint4(0, 0, 0, 0);
  } else {
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = col + k < D ? to_f32(row[col + k]) : 0.f;
    pack(f, r);                     // exact: the values are of type T
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ row, int col, int D, const float (&f)[8]) {
  if (VEC) {
    if (col >= D) return;
    Vec8<T> r;
    pack(f, r);
#pragma unroll
    for (int i = 0; i < Vec8<T>::Q; ++i) *(reinterpret_cast<uint4*>(row + col) + i) = r.q[i];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (col + k < D) row[col + k] = from_f32<T>(f[k]);
  }
}

// Weight or bias columns [col, col + 8) as fp32; `fp32`: stored as fp32, else as T.
template <typename T>
__device__ __forceinline__ void load_param8(const void* p, int fp32, int col, int D, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int c = col + k;
    f[k] = c >= D ? 0.f : fp32 ? __ldg(static_cast<const float*>(p) + c) : to_f32(static_cast<const T*>(p)[c]);
  }
}

// ---- the dropout generator -------------------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011).  One call gives
// the eight 16-bit numbers of eight columns: counter = (group low, group high, offset, site), key = seed, where
// group = row * ceil(D / 8) + column / 8.  16 bits set a drop probability to the nearest 1 / 65536 and halve the
// generator's work an element against 32, which keeps it below the memory time.
struct Generator {
  uint32_t k0, k1, offset, site;
};

__device__ __forceinline__ uint4 philox(const Generator& g, uint64_t group) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = g.offset, c3 = g.site;
  uint32_t k0 = g.k0, k1 = g.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ Generator load_generator(const int64_t* rng, uint32_t site) {
  const uint64_t seed = (uint64_t)__ldg(reinterpret_cast<const long long*>(rng));
  const uint64_t offset = (uint64_t)__ldg(reinterpret_cast<const long long*>(rng) + 1);
  return Generator{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, site};
}

// bit j: element j of the group is kept (its 16-bit number is not below the threshold)
__device__ __forceinline__ uint32_t keep_bits(const Generator& g, uint64_t group, uint32_t threshold) {
  const uint4 r = philox(g, group);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if ((w[k] & 0xFFFFu) >= threshold) bits |= 1u << (2 * k);
    if ((w[k] >> 16) >= threshold) bits |= 2u << (2 * k);
  }
  return bits;
}

// ---- a row's warps ---------------------------------------------------------------------------------------------------
constexpr int kMaxRowWarps = 8;

// Sums of two values over the W warps of a row, the same in every lane and in the same order on every run.  `slot`
// points at this row group's [2][kMaxRowWarps] exchange; it alternates, so one barrier a reduction is enough: a warp
// that writes slot k again has passed the barrier behind the reads of it.
struct RowGroup {
  int W, sub, bar;
  float2* slot;
  int phase;
};

__device__ __forceinline__ void row_sum2(RowGroup& g, float& a, float& b) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (g.W > 1) {
    float2* s = g.slot + g.phase * kMaxRowWarps;
    g.phase ^= 1;
    if ((threadIdx.x & 31) == 0) s[g.sub] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(g.bar), "r"(g.W * 32) : "memory");
    a = 0.f;
    b = 0.f;
    for (int i = 0; i < g.W; ++i) {
      const float2 v = s[i];
      a += v.x;
      b += v.y;
    }
  }
}

__device__ __forceinline__ bool padding_row(const RowArgs& a, int row) {
  if (a.lengths == nullptr) return false;
  const int b = row / a.T;
  return row - b * a.T >= __ldg(a.lengths + b);
}

// LayerNorm forward; DROP: of h = residual + dropout(x), which is stored too.  W warps a row, NV vectors of eight
// columns a lane: a row stays in registers between the two passes of its statistics.
template <typename T, int NV, bool VEC, bool DROP>
__global__ void __launch_bounds__(256) ln_fwd_kernel(RowArgs a) {
  __shared__ float2 exchange[8][2 * kMaxRowWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.W, R = (blockDim.x >> 5) / W;
  const int group = warp / W;
  RowGroup rg{W, warp - group * W, 1 + group, exchange[group], 0};
  const int D = a.D;
  int col[NV];
  float wv[NV][8], bv[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = ((i * W + rg.sub) * 32 + lane) * 8;
    load_param8<T>(a.weight, a.param_fp32, col[i], D, wv[i]);
    load_param8<T>(a.bias, a.param_fp32, col[i], D, bv[i]);
  }
  Generator gen{};
  if (DROP) gen = load_generator(a.rng, a.site);
  const float inv_d = 1.0f / D;
  for (int64_t row = (int64_t)blockIdx.x * R + group; row < a.M; row += (int64_t)gridDim.x * R) {
    T* y = static_cast<T*>(a.y) + row * D;
    T* h = DROP ? static_cast<T*>(a.h_out) + row * D : nullptr;
    const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
    const T* res = DROP ? static_cast<const T*>(a.residual) + row * a.ld_res : nullptr;
    const bool pad = padding_row(a, (int)row);
    float v[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Vec8<T> r;
      if (DROP) {
        load8<T, VEC>(res, col[i], D, r);
        unpack(r, v[i]);
        if (!pad) {
          float f[8];
          load8<T, VEC>(x, col[i], D, r);
          unpack(r, f);
          const uint32_t keep = keep_bits(gen, (uint64_t)row * a.groups + (col[i] >> 3), a.threshold);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (keep >> k & 1) v[i][k] = fmaf(f[k], a.factor, v[i][k]);
        }
        store8<T, VEC>(h, col[i], D, v[i]);
      } else if (!pad) {
        load8<T, VEC>(x, col[i], D, r);
        unpack(r, v[i]);
      }
    }
    if (pad) {
      const float zero[8] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) store8<T, VEC>(y, col[i], D, zero);
      continue;
    }
    float s = 0.f, none = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) s += col[i] + k < D ? v[i][k] : 0.f;
    row_sum2(rg, s, none);
    const float mean = s * inv_d;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float d = col[i] + k < D ? v[i][k] - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    row_sum2(rg, sq, none);
    const float rstd = rsqrtf(fmaf(sq, inv_d, a.eps));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = fmaf((v[i][k] - mean) * rstd, wv[i][k], bv[i][k]);
      store8<T, VEC>(y, col[i], D, o);
    }
  }
}

// LayerNorm backward; the row's statistics are formed again from x, which has to be read anyway.  With d = x - m the
// sums are S0 = sum g and, once m is known, S1 = sum d^2 and S2 = sum g d: dx = r (g - S0 / D - d r^2 S2 / D).
// DROP: x is the stored h, the incoming gradient dh of h joins dx, and dropout's gradient is written beside it.  Each
// lane keeps the running sums of its columns' dw and db over all rows of its warp; the CTA adds its row groups in
// order and leaves one partial row, so no sum depends on the order of arrival.
template <typename T, int NV, bool VEC, bool DROP>
__global__ void __launch_bounds__(256) ln_bwd_kernel(RowArgs a) {
  __shared__ float2 exchange[8][2 * kMaxRowWarps];
  extern __shared__ float combine[];               // [2][D] with more than one row group a CTA
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.W, R = (blockDim.x >> 5) / W;
  const int group = warp / W;
  RowGroup rg{W, warp - group * W, 1 + group, exchange[group], 0};
  const int D = a.D;
  int col[NV];
  float wv[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = ((i * W + rg.sub) * 32 + lane) * 8;
    load_param8<T>(a.weight, a.param_fp32, col[i], D, wv[i]);
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[i][k] = db[i][k] = 0.f;
  }
  Generator gen{};
  if (DROP) gen = load_generator(a.rng, a.site);
  const float inv_d = 1.0f / D;
  for (int64_t row = (int64_t)blockIdx.x * R + group; row < a.M; row += (int64_t)gridDim.x * R) {
    T* dx = static_cast<T*>(a.dx) + row * D;
    T* dres = DROP ? static_cast<T*>(a.dres) + row * D : nullptr;
    const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
    const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
    const T* dh = DROP && a.dh ? static_cast<const T*>(a.dh) + row * a.ld_dh : nullptr;
    if (padding_row(a, (int)row)) {
      const float zero[8] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        store8<T, VEC>(dx, col[i], D, zero);
        if (DROP) {
          float f[8] = {};
          if (dh) {
            Vec8<T> r;
            load8<T, VEC>(dh, col[i], D, r);
            unpack(r, f);
          }
          store8<T, VEC>(dres, col[i], D, f);
        }
      }
      continue;
    }
    Vec8<T> xr[NV], gr[NV], hr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      load8<T, VEC>(x, col[i], D, xr[i]);
      load8<T, VEC>(dy, col[i], D, gr[i]);
      if (DROP && dh) load8<T, VEC>(dh, col[i], D, hr[i]);
    }
    float s = 0.f, s0 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[8], g[8];
      unpack(xr[i], f);
      unpack(gr[i], g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {                // columns past D are zero in x and dy
        s += f[k];
        s0 = fmaf(g[k], wv[i][k], s0);
      }
    }
    row_sum2(rg, s, s0);
    const float mean = s * inv_d;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[8], g[8];
      unpack(xr[i], f);
      unpack(gr[i], g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float d = col[i] + k < D ? f[k] - mean : 0.f;
        s1 = fmaf(d, d, s1);
        s2 = fmaf(g[k] * wv[i][k], d, s2);
      }
    }
    row_sum2(rg, s1, s2);
    const float rstd = rsqrtf(fmaf(s1, inv_d, a.eps));
    const float c1 = s0 * inv_d, c2 = rstd * rstd * (s2 * inv_d);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[8], g[8], o[8];
      unpack(xr[i], f);
      unpack(gr[i], g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float d = f[k] - mean;
        o[k] = rstd * (fmaf(g[k], wv[i][k], -c1) - d * c2);
        dw[i][k] = fmaf(g[k], d * rstd, dw[i][k]);
        db[i][k] += g[k];
      }
      if (DROP) {
        if (dh) {
          unpack(hr[i], f);
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] += f[k];
        }
        store8<T, VEC>(dres, col[i], D, o);
        const uint32_t keep = keep_bits(gen, (uint64_t)row * a.groups + (col[i] >> 3), a.threshold);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = keep >> k & 1 ? o[k] * a.factor : 0.f;
      }
      store8<T, VEC>(dx, col[i], D, o);
    }
  }
  float* out = a.partials + (int64_t)blockIdx.x * 2 * D;
  for (int g = 0; g < R; ++g) {
    if (R > 1) __syncthreads();
    if (group != g) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = col[i] + k;
        if (c >= D) continue;
        float sw = dw[i][k], sb = db[i][k];
        if (g > 0) {
          sw += combine[c];
          sb += combine[D + c];
        }
        if (g + 1 < R) {
          combine[c] = sw;
          combine[D + c] = sb;
        } else {
          out[c] = sw;
          out[D + c] = sb;
        }
      }
  }
}

// dw and db: the sums over the CTAs' partial rows, in a fixed order.  32 columns a CTA, 8 warps striding the rows.
template <typename T>
__global__ void __launch_bounds__(256) ln_param_grad_kernel(const float* __restrict__ partials, int rows, int D,
                                                            void* dweight, void* dbias, int fp32) {
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;            // column of [dw | db]
  float s = 0.f;
  if (c < 2 * D)
    for (int r = warp; r < rows; r += 8) s += __ldg(partials + (int64_t)r * 2 * D + c);
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < 2 * D) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += part[i][lane];
    void* dst = c < D ? dweight : dbias;
    const int k = c < D ? c : c - D;
    if (fp32)
      static_cast<float*>(dst)[k] = s;
    else
      static_cast<T*>(dst)[k] = from_f32<T>(s);
  }
}

// out = residual + dropout(x), one group of eight columns a thread.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(RowArgs a, int64_t n) {
  const Generator gen = load_generator(a.rng, a.site);
  const int D = a.D;
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
    const int64_t r = i / a.groups;
    const int col = (int)(i - r * a.groups) * 8;
    const int64_t row = r;
    float v[8] = {};
    Vec8<T> q;
    if (a.residual) {
      load8<T, VEC>(static_cast<const T*>(a.residual) + row * a.ld_res, col, D, q);
      unpack(q, v);
    }
    if (!padding_row(a, (int)row)) {
      float f[8];
      load8<T, VEC>(static_cast<const T*>(a.x) + row * a.ld_x, col, D, q);
      unpack(q, f);
      const uint32_t keep = keep_bits(gen, (uint64_t)row * a.groups + (col >> 3), a.threshold);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (keep >> k & 1) v[k] = fmaf(f[k], a.factor, v[k]);
    }
    store8<T, VEC>(static_cast<T*>(a.y) + row * D, col, D, v);
  }
}

// A row's warps and vectors a lane: the fewest warps that hold the row in four vectors (32 columns) a lane.
struct RowShape {
  int W, NV, warps;
};
RowShape row_shape(int D) {
  const int vec = (D + 255) / 256;                 // vectors of 256 columns a warp
  RowShape s;
  s.W = 1;
  while (s.W * 4 < vec) s.W *= 2;
  s.NV = (vec + s.W - 1) / s.W;
  s.NV = s.NV == 3 ? 4 : s.NV;
  s.warps = 8;
  return s;
}

bool vec_ok(const RowArgs& a, int size) {
  const int per = 16 / size;
  const int64_t lds[] = {a.ld_x, a.ld_dy, a.ld_dh, a.ld_res};
  const void* ptrs[] = {a.x, a.dy, a.dh, a.residual, a.y, a.h_out, a.dx, a.dres};
  if (a.D % 8) return false;
  for (int64_t l : lds)
    if (l % per) return false;
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  return true;
}

template <typename T, int NV, bool VEC, bool DROP>
int launch_fwd(const RowArgs& a, const RowShape& s, cudaStream_t stream) {
  const int R = s.warps / s.W;
  const int64_t want = (a.M + R - 1) / R;
  const int grid = (int)(want < 4 * device_sm_count() ? want : 4 * device_sm_count());
  ln_fwd_kernel<T, NV, VEC, DROP><<<grid, s.warps * 32, 0, stream>>>(a);
  return (int)cudaGetLastError();
}

template <typename T, int NV, bool VEC, bool DROP>
int launch_bwd(const RowArgs& a, const RowShape& s, cudaStream_t stream) {
  const int R = s.warps / s.W;
  const size_t smem = R > 1 ? (size_t)2 * a.D * sizeof(float) : 0;
  ln_bwd_kernel<T, NV, VEC, DROP><<<(int)a.partial_rows, s.warps * 32, smem, stream>>>(a);
  if (cudaError_t e = cudaGetLastError()) return (int)e;
  return 0;
}

template <typename T, bool VEC, bool DROP>
int launch_rows(const RowArgs& a, bool bwd, cudaStream_t stream) {
  const RowShape s = row_shape(a.D);
  RowArgs b = a;
  b.W = s.W;
  switch (s.NV) {
    case 1: return bwd ? launch_bwd<T, 1, VEC, DROP>(b, s, stream) : launch_fwd<T, 1, VEC, DROP>(b, s, stream);
    case 2: return bwd ? launch_bwd<T, 2, VEC, DROP>(b, s, stream) : launch_fwd<T, 2, VEC, DROP>(b, s, stream);
    default: return bwd ? launch_bwd<T, 4, VEC, DROP>(b, s, stream) : launch_fwd<T, 4, VEC, DROP>(b, s, stream);
  }
}

template <typename T>
int launch_typed(const RowArgs& a, int op, cudaStream_t stream) {
  const bool vec = vec_ok(a, sizeof(T));
  if (op == kRowDropout) {
    // the grid's thread index counts groups in 64 bits
    const int64_t n = a.M * a.groups;
    const int64_t want = (n + 255) / 256;
    const int64_t most = 16 * (int64_t)device_sm_count();
    const int grid = (int)(want < most ? want : most);
    if (vec)
      dropout_kernel<T, true><<<grid, 256, 0, stream>>>(a, n);
    else
      dropout_kernel<T, false><<<grid, 256, 0, stream>>>(a, n);
    return (int)cudaGetLastError();
  }
  const bool drop = op == kRowDropNorm || op == kRowDropNormGrad, bwd = op == kRowNormGrad || op == kRowDropNormGrad;
  if (a.M > 0) {
    const int rc = drop ? (vec ? launch_rows<T, true, true>(a, bwd, stream) : launch_rows<T, false, true>(a, bwd, stream))
                        : (vec ? launch_rows<T, true, false>(a, bwd, stream)
                               : launch_rows<T, false, false>(a, bwd, stream));
    if (rc) return rc;
  }
  if (bwd) {
    ln_param_grad_kernel<T><<<(2 * a.D + 31) / 32, 256, 0, stream>>>(a.partials, (int)a.partial_rows, a.D, a.dweight,
                                                                     a.dbias, a.param_fp32);
    return (int)cudaGetLastError();
  }
  return 0;
}

}  // namespace rows_impl

int row_partial_rows(int64_t M, int D) {
  const rows_impl::RowShape s = rows_impl::row_shape(D);
  const int R = s.warps / s.W;
  const int64_t want = (M + R - 1) / R;
  return (int)(want < 2 * device_sm_count() ? want : 2 * device_sm_count());
}

int launch_row_op(const RowArgs& args, int op, int dtype, cudaStream_t stream) {
  using namespace rows_impl;
  switch (dtype) {
    case 0: return launch_typed<__nv_bfloat16>(args, op, stream);
    case 1: return launch_typed<__half>(args, op, stream);
    default: return launch_typed<float>(args, op, stream);
  }
}

}  // namespace gsn
