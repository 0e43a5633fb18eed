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
#include <algorithm>

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

// fp32 pairs, two lanes an instruction (sm_100)
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ void unpack(const Vec8<__nv_bfloat16>& r, float2 (&f)[4]) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = make_float2(bf16lo_to_f32(w[k]), bf16hi_to_f32(w[k]));
}
__device__ __forceinline__ void unpack(const Vec8<__half>& r, float2 (&f)[4]) {
  const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
}
__device__ __forceinline__ void unpack(const Vec8<float>& r, float2 (&f)[4]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    f[2 * k] = make_float2(__uint_as_float(r.q[k].x), __uint_as_float(r.q[k].y));
    f[2 * k + 1] = make_float2(__uint_as_float(r.q[k].z), __uint_as_float(r.q[k].w));
  }
}
__device__ __forceinline__ void pack(const float2 (&f)[4], Vec8<__nv_bfloat16>& r) {
  r.q[0] = make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y),
                      pack_bf16x2(f[3].x, f[3].y));
}
__device__ __forceinline__ void pack(const float2 (&f)[4], Vec8<__half>& r) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __half2 h = __float22half2_rn(f[k]);
    w[k] = *reinterpret_cast<const uint32_t*>(&h);
  }
  r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack(const float2 (&f)[4], Vec8<float>& r) {
#pragma unroll
  for (int k = 0; k < 2; ++k)
    r.q[k] = make_uint4(__float_as_uint(f[2 * k].x), __float_as_uint(f[2 * k].y), __float_as_uint(f[2 * k + 1].x),
                        __float_as_uint(f[2 * k + 1].y));
}

// the same as single values (the CTC kernels)
template <typename T>
__device__ __forceinline__ void unpack(const Vec8<T>& r, float (&f)[8]) {
  float2 p[4];
  unpack(r, p);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = p[k].x;
    f[2 * k + 1] = p[k].y;
  }
}
template <typename T>
__device__ __forceinline__ void pack(const float (&f)[8], Vec8<T>& r) {
  const float2 p[4] = {{f[0], f[1]}, {f[2], f[3]}, {f[4], f[5]}, {f[6], f[7]}};
  pack(p, r);
}

// A warp's block of 256 columns: lane l holds eight of them.  VEC (rows aligned to 16 bytes, D % 8 == 0): of a 16-bit
// type columns 8 l .. 8 l + 7, of fp32 columns 4 l .. 4 l + 3 and 128 further on: one and two 16-byte words, a warp's
// words without a gap.  Otherwise columns l + 32 k, so that single elements still make whole 32-byte sectors.
template <typename T, bool VEC>
__device__ __forceinline__ int column(int base, int lane, int k) {
  if (!VEC) return base + k * 32 + lane;
  return sizeof(T) == 2 ? base + lane * 8 + k : base + (k >> 2) * 128 + lane * 4 + (k & 3);
}
// the first column of 16-byte word q (VEC)
template <typename T>
__device__ __forceinline__ int word_column(int base, int lane, int q) { return column<T, true>(base, lane, q * 4); }

// columns past D read as zero
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, int base, int lane, int D, Vec8<T>& r) {
  if (VEC) {
#pragma unroll
    for (int q = 0; q < Vec8<T>::Q; ++q) {
      const int col = word_column<T>(base, lane, q);
      r.q[q] = col < D ? __ldg(reinterpret_cast<const uint4*>(row + col)) : make_uint4(0, 0, 0, 0);
    }
  } else {
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int col = column<T, VEC>(base, lane, k);
      f[k] = col < D ? to_f32(row[col]) : 0.f;
    }
    pack(f, r);                     // exact: the values are of type T
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ row, int base, int lane, int D, const float2 (&f)[4]) {
  if (VEC) {
    Vec8<T> r;
    pack(f, r);
#pragma unroll
    for (int q = 0; q < Vec8<T>::Q; ++q) {
      const int col = word_column<T>(base, lane, q);
      if (col < D) *reinterpret_cast<uint4*>(row + col) = r.q[q];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int col = column<T, VEC>(base, lane, k);
      if (col < D) row[col] = from_f32<T>(k & 1 ? f[k / 2].y : f[k / 2].x);
    }
  }
}

// The lane's columns of weight or bias as fp32; `fp32`: stored as fp32, else as T.
template <typename T, bool VEC>
__device__ __forceinline__ void load_param8(const void* p, int fp32, int base, int lane, int D, float2 (&f)[4]) {
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int c = column<T, VEC>(base, lane, k);
    v[k] = c >= D ? 0.f : fp32 ? __ldg(static_cast<const float*>(p) + c) : to_f32(static_cast<const T*>(p)[c]);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = make_float2(v[2 * k], v[2 * k + 1]);
}

// v where the columns of pair k are inside the row, else 0
template <typename T, bool VEC>
__device__ __forceinline__ float2 inside(float v, int base, int lane, int k, int D) {
  if (VEC) return both(column<T, true>(base, lane, 2 * k) < D ? v : 0.f);
  return make_float2(column<T, VEC>(base, lane, 2 * k) < D ? v : 0.f, column<T, VEC>(base, lane, 2 * k + 1) < D ? v : 0.f);
}

__device__ __forceinline__ void copy16(void* smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(gmem) : "memory");
}

// Rows under way: each thread copies the 16-byte words that it will itself read, some rows ahead, so the loads need
// neither registers nor a barrier.  TENSORS inputs of NV blocks a lane; slots [stage][tensor][block][word][thread].
constexpr int kRowThreads = 256;

template <typename T, int NV, int TENSORS>
struct Ring {
  static constexpr int Q = Vec8<T>::Q, WORDS = TENSORS * NV * Q, STAGE = WORDS * kRowThreads;
  uint4* slots;                                    // this thread's first, in shared memory
  static __device__ __forceinline__ constexpr int at(int tensor, int i, int q) {
    return ((tensor * NV + i) * Q + q) * kRowThreads;
  }
  __device__ __forceinline__ void fetch(int stage, int tensor, int i, const T* row, int base, int lane, int D) const {
    uint4* dst = slots + stage * STAGE;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int col = word_column<T>(base, lane, q);
      if (col < D) copy16(dst + at(tensor, i, q), row + col);
    }
  }
  __device__ __forceinline__ void read(int stage, int tensor, int i, Vec8<T>& r) const {
    const uint4* src = slots + stage * STAGE;
#pragma unroll
    for (int q = 0; q < Q; ++q) r.q[q] = src[at(tensor, i, q)];
  }
  // columns past D are never copied: zeros, once
  __device__ __forceinline__ void clear(int stages) const {
    for (int i = 0; i < stages * WORDS; ++i) slots[i * kRowThreads] = make_uint4(0, 0, 0, 0);
  }
};

template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// ---- the dropout generator -------------------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011).  One call gives
// the eight 16-bit numbers of eight columns: counter = (group low, group high, offset, site), key = seed, where
// group = row * ceil(D / 8) + column / 8.  16 bits set a drop probability to the nearest 1 / 65536 and halve the
// generator's work an element against 32, which keeps it below the memory time.
struct Generator {
  uint32_t k0, k1, offset, site;
};

__device__ __forceinline__ Generator load_generator(const int64_t* rng, uint32_t site) {
  const uint64_t seed = (uint64_t)__ldg(reinterpret_cast<const long long*>(rng));
  const uint64_t offset = (uint64_t)__ldg(reinterpret_cast<const long long*>(rng) + 1);
  return Generator{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, site};
}

// the eight numbers of N groups at a time, round by round: the keys of a round are formed once
template <int N>
__device__ __forceinline__ void philox(const Generator& g, const uint64_t (&group)[N], uint4 (&out)[N]) {
  uint32_t c0[N], c1[N], c2[N], c3[N], k0 = g.k0, k1 = g.k1;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    c0[n] = (uint32_t)group[n];
    c1[n] = (uint32_t)(group[n] >> 32);
    c2[n] = g.offset;
    c3[n] = g.site;
  }
#pragma unroll
  for (int i = 0; i < 10; ++i) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint64_t a = (uint64_t)0xD2511F53u * c0[n], b = (uint64_t)0xCD9E8D57u * c2[n];
      c0[n] = (uint32_t)(b >> 32) ^ c1[n] ^ k0;
      c1[n] = (uint32_t)b;
      c2[n] = (uint32_t)(a >> 32) ^ c3[n] ^ k1;
      c3[n] = (uint32_t)a;
    }
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
#pragma unroll
  for (int n = 0; n < N; ++n) out[n] = make_uint4(c0[n], c1[n], c2[n], c3[n]);
}

// The kept ones of a group's eight elements in their order, the others 0 (chosen, not multiplied: a dropped infinity is
// gone).  An element is kept where its 16-bit number is not below the threshold, given shifted up by 16.
__device__ __forceinline__ void keep8(const uint4& r, uint32_t threshold16, float2 (&f)[4]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[k].x = (w[k] << 16) >= threshold16 ? f[k].x : 0.f;
    f[k].y = w[k] >= threshold16 ? f[k].y : 0.f;
  }
}

// the same as bits, number j in bit j
__device__ __forceinline__ uint32_t keep_bits(const uint4& r, uint32_t threshold16) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    bits |= (w[k] << 16) >= threshold16 ? 1u << (2 * k) : 0u;
    bits |= w[k] >= threshold16 ? 2u << (2 * k) : 0u;
  }
  return bits;
}

// Which of a lane's elements of NV blocks are kept.  The generator's groups are neighbours, so a 16-bit type's eight
// elements a block are a group; fp32's two halves belong to two groups and single elements to eight, drawn by other
// lanes: there the answers travel as bits, 8 i + k.
template <typename T, int NV, bool VEC>
struct Kept {
  static constexpr bool OWN = VEC && sizeof(T) == 2;
  uint4 drawn[OWN ? NV : 1];
  uint32_t bits;

  __device__ __forceinline__ void draw(const Generator& g, uint64_t row_group, const int (&base)[NV], int lane,
                                       uint32_t threshold16) {
    static_assert(NV <= 4, "eight bits a block in one word");
    uint64_t group[NV];
    uint4 r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) group[i] = row_group + (base[i] >> 3) + lane;
    philox(g, group, r);
    if constexpr (OWN) {
#pragma unroll
      for (int i = 0; i < NV; ++i) drawn[i] = r[i];
    } else {
      to_bits(r, lane, threshold16);
    }
  }

  __device__ __forceinline__ void to_bits(const uint4 (&r)[NV], int lane, uint32_t threshold16) {
    uint32_t own = 0;
    bits = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) own |= keep_bits(r[i], threshold16) << (8 * i);
    if constexpr (VEC) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {                // columns base + 128 q + 4 l: group 16 q + l / 2, its half l % 2
        const uint32_t w = __shfl_sync(0xffffffffu, own, 16 * q + (lane >> 1)) >> (4 * (lane & 1));
        bits |= (w & 0x0F0F0F0Fu) << (4 * q);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {                // column base + 32 k + lane: group 4 k + lane / 8, its bit lane % 8
        const uint32_t w = __shfl_sync(0xffffffffu, own, 4 * k + (lane >> 3)) >> (lane & 7);
        bits |= (w & 0x01010101u) << k;
      }
    }
  }

  __device__ __forceinline__ void apply(int i, uint32_t threshold16, float2 (&f)[4]) const {
    if constexpr (OWN) {
      keep8(drawn[i], threshold16, f);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f[k].x = bits & (1u << (8 * i + 2 * k)) ? f[k].x : 0.f;
        f[k].y = bits & (2u << (8 * i + 2 * k)) ? f[k].y : 0.f;
      }
    }
  }
};

// ---- a row's warps ---------------------------------------------------------------------------------------------------
constexpr int kMaxRowWarps = 8;

// Sums over the W warps of a row, the same in every lane and in the same order on every run.  `slot` points at this row
// group's exchange, [2 phases][2 values][8 warps], zeros where there is no warp; the phases alternate, so one barrier a
// reduction is enough: a warp that writes a phase again has passed the barrier behind the reads of it.
struct RowGroup {
  int W, sub, bar;
  float* slot;
  int phase;
};

template <int N>
__device__ __forceinline__ void row_sums(RowGroup& g, float (&v)[N]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (g.W > 1) {
    float* s = g.slot + g.phase;
    g.phase ^= 2 * kMaxRowWarps;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[i * kMaxRowWarps + g.sub] = v[i];
    asm volatile("bar.sync %0, %1;" ::"r"(g.bar), "r"(g.W * 32) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float4 lo = *reinterpret_cast<const float4*>(s + i * kMaxRowWarps);
      v[i] = (lo.x + lo.y) + (lo.z + lo.w);
      if (g.W > 4) {
        const float4 hi = *reinterpret_cast<const float4*>(s + i * kMaxRowWarps + 4);
        v[i] += (hi.x + hi.y) + (hi.z + hi.w);
      }
    }
  }
}

// The sum of a lane's pairs in four chains: a single one would wait for its own additions.
template <int NV, typename F>
__device__ __forceinline__ float2 lane_sum(F term) {
  float2 c[4] = {both(0.f), both(0.f), both(0.f), both(0.f)};
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = term(i, k, c[k]);
  return add2(add2(c[0], c[1]), add2(c[2], c[3]));
}

// row / T by a multiplication (the launcher sets the factor), for row < 2^31
__device__ __forceinline__ bool padding_row(const RowArgs& a, uint32_t row) {
  if (a.lengths == nullptr) return false;
  const uint32_t b = (__umulhi(a.div_factor, row) + row) >> a.div_shift;
  return (int)(row - b * (uint32_t)a.T) >= __ldg(a.lengths + b);
}

// Rows under way a warp: as many as leave two CTAs an SM (one where a lane holds 32 columns of fp32)
__host__ __device__ constexpr int ring_stages(int words) { return words <= 6 ? 4 : words <= 8 ? 3 : 2; }

// LayerNorm forward; DROP: of h = residual + dropout(x), which is stored too.  W warps a row, NV blocks of 256 columns
// a warp: a row stays in registers between the two passes of its statistics, its weights for all rows of the warp.
template <typename T, int NV, bool VEC, bool DROP>
__global__ void __launch_bounds__(kRowThreads, NV < 4 ? 2 : 1) ln_fwd_kernel(RowArgs a) {
  __shared__ __align__(16) float exchange[8][4 * kMaxRowWarps];
  extern __shared__ uint4 ring_slots[];
  constexpr int TENSORS = DROP ? 2 : 1, S = ring_stages(Ring<T, NV, TENSORS>::WORDS);
  const Ring<T, NV, TENSORS> ring{ring_slots + threadIdx.x};
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.W, R = (kRowThreads >> 5) / W;
  const int group = warp / W;
  (&exchange[0][0])[threadIdx.x] = 0.f;
  RowGroup rg{W, warp - group * W, 1 + group, exchange[group], 0};
  const int D = a.D;
  int base[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) base[i] = (i * W + rg.sub) * 256;
  const uint32_t M = (uint32_t)a.M, stride = gridDim.x * R, first = blockIdx.x * R + group;
  uint32_t ahead = first, pads = 0;                // the row to fetch next; bit s: stage s holds a padding row
  const T* x_ahead = static_cast<const T*>(a.x) + first * a.ld_x;
  const T* res_ahead = DROP ? static_cast<const T*>(a.residual) + first * a.ld_res : nullptr;
  auto fetch = [&](int stage) {
    pads &= ~(1u << stage);
    if (ahead < M) {
      const bool pad = padding_row(a, ahead);
      pads |= (pad ? 1u : 0u) << stage;
      if (VEC) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (!pad && !(DROP && a.drop_all)) ring.fetch(stage, 0, i, x_ahead, base[i], lane, D);
          if (DROP) ring.fetch(stage, 1, i, res_ahead, base[i], lane, D);
        }
        x_ahead += stride * a.ld_x;
        if (DROP) res_ahead += stride * a.ld_res;
      }
    }
    ahead += stride;
    if (VEC) copies_commit();
  };
  if (VEC) ring.clear(S);
#pragma unroll
  for (int s = 0; s + 1 < S; ++s) fetch(s);
  __syncthreads();                                 // the exchange is cleared
  float2 wv[NV][4], bv[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_param8<T, VEC>(a.weight, a.param_fp32, base[i], lane, D, wv[i]);
    load_param8<T, VEC>(a.bias, a.param_fp32, base[i], lane, D, bv[i]);
  }
  Generator gen{};
  if (DROP) gen = load_generator(a.rng, a.site);
  const float inv_d = 1.0f / D;
  int stage = 0;
  for (uint32_t row = first; row < M; row += stride) {
    T* y = static_cast<T*>(a.y) + (int64_t)row * D;
    fetch(stage == 0 ? S - 1 : stage - 1);
    const bool pad = pads >> stage & 1;
    if (VEC) copies_wait<S - 1>();
    float2 v[NV][4];
    auto input = [&](int tensor, const void* p, int64_t ld, int i, float2 (&f)[4]) {
      Vec8<T> r;
      if (VEC)
        ring.read(stage, tensor, i, r);
      else
        load8<T, VEC>(static_cast<const T*>(p) + (int64_t)row * ld, base[i], lane, D, r);
      unpack(r, f);
    };
    if (DROP) {
      const bool add = !pad && !a.drop_all;
      Kept<T, NV, VEC> kept;
      if (add) kept.draw(gen, (uint64_t)row * a.groups, base, lane, a.threshold << 16);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        input(1, a.residual, a.ld_res, i, v[i]);
        if (add) {
          float2 f[4];
          input(0, a.x, a.ld_x, i, f);
          kept.apply(i, a.threshold << 16, f);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[i][k] = ffma2(f[k], both(a.factor), v[i][k]);
        }
        store8<T, VEC>(static_cast<T*>(a.h_out) + (int64_t)row * D, base[i], lane, D, v[i]);
      }
    } else if (!pad) {
#pragma unroll
      for (int i = 0; i < NV; ++i) input(0, a.x, a.ld_x, i, v[i]);
    }
    stage = stage + 1 == S ? 0 : stage + 1;
    if (pad) {
      const float2 zero[4] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) store8<T, VEC>(y, base[i], lane, D, zero);
      continue;
    }
    // columns past D are zero
    float2 acc = lane_sum<NV>([&](int i, int k, float2 c) { return add2(c, v[i][k]); });
    float sum[1] = {acc.x + acc.y};
    row_sums(rg, sum);
    const float mean = sum[0] * inv_d;
    acc = lane_sum<NV>([&](int i, int k, float2 c) {
      v[i][k] = add2(v[i][k], inside<T, VEC>(-mean, base[i], lane, k, D));
      return ffma2(v[i][k], v[i][k], c);
    });
    sum[0] = acc.x + acc.y;
    row_sums(rg, sum);
    const float rstd = rsqrtf(fmaf(sum[0], inv_d, a.eps));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float2 o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = ffma2(mul2(v[i][k], both(rstd)), wv[i][k], bv[i][k]);
      store8<T, VEC>(y, base[i], lane, D, o);
    }
  }
}

// LayerNorm backward; the row's statistics are formed again from x, which has to be read anyway.  With d = x - m the
// sums are S0 = sum g and, once m is known, S1 = sum d^2 and S2 = sum g d: dx = r (g - S0 / D - d r^2 S2 / D).
// DROP: x is the stored h, the incoming gradient dh of h joins dx, and dropout's gradient is written beside it.  Each
// lane keeps the running sums of its columns' dw and db over all rows of its warp; the CTA adds its row groups in
// order and leaves one partial row, so no sum depends on the order of arrival.
template <typename T, int NV, bool VEC, bool DROP>
__global__ void __launch_bounds__(kRowThreads, NV < 4 ? 2 : 1) ln_bwd_kernel(RowArgs a) {
  __shared__ __align__(16) float exchange[8][4 * kMaxRowWarps];
  extern __shared__ uint4 ring_slots[];            // the ring; at the end [2][D], the CTA's sums
  kernel_let_next();                               // the sums' kernel stands ready
  constexpr int TENSORS = DROP ? 3 : 2, S = ring_stages(Ring<T, NV, TENSORS>::WORDS);
  const Ring<T, NV, TENSORS> ring{ring_slots + threadIdx.x};
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.W, R = (kRowThreads >> 5) / W;
  const int group = warp / W;
  (&exchange[0][0])[threadIdx.x] = 0.f;
  RowGroup rg{W, warp - group * W, 1 + group, exchange[group], 0};
  const int D = a.D;
  int base[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) base[i] = (i * W + rg.sub) * 256;
  const uint32_t M = (uint32_t)a.M, stride = gridDim.x * R, first = blockIdx.x * R + group;
  uint32_t ahead = first, pads = 0;                // the row to fetch next; bit s: stage s holds a padding row
  const T* x_ahead = static_cast<const T*>(a.x) + first * a.ld_x;
  const T* dy_ahead = static_cast<const T*>(a.dy) + first * a.ld_dy;
  const T* dh_ahead = DROP && a.dh ? static_cast<const T*>(a.dh) + first * a.ld_dh : nullptr;
  auto fetch = [&](int stage) {
    pads &= ~(1u << stage);
    if (ahead < M) {
      const bool pad = padding_row(a, ahead);
      pads |= (pad ? 1u : 0u) << stage;
      if (VEC) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (!pad) {
            ring.fetch(stage, 0, i, x_ahead, base[i], lane, D);
            ring.fetch(stage, 1, i, dy_ahead, base[i], lane, D);
          }
          if (DROP && dh_ahead) ring.fetch(stage, TENSORS - 1, i, dh_ahead, base[i], lane, D);
        }
        x_ahead += stride * a.ld_x;
        dy_ahead += stride * a.ld_dy;
        if (DROP && dh_ahead) dh_ahead += stride * a.ld_dh;
      }
    }
    ahead += stride;
    if (VEC) copies_commit();
  };
  if (VEC) ring.clear(S);                          // and zeros stand in for a missing dh
#pragma unroll
  for (int s = 0; s + 1 < S; ++s) fetch(s);
  __syncthreads();                                 // the exchange is cleared
  float2 wv[NV][4], dw[NV][4], db[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_param8<T, VEC>(a.weight, a.param_fp32, base[i], lane, D, wv[i]);
#pragma unroll
    for (int k = 0; k < 4; ++k) dw[i][k] = db[i][k] = both(0.f);
  }
  Generator gen{};
  if (DROP) gen = load_generator(a.rng, a.site);
  const float inv_d = 1.0f / D;
  int stage = 0;
  for (uint32_t row = first; row < M; row += stride) {
    T* dx = static_cast<T*>(a.dx) + (int64_t)row * D;
    T* dres = DROP ? static_cast<T*>(a.dres) + (int64_t)row * D : nullptr;
    fetch(stage == 0 ? S - 1 : stage - 1);
    const bool pad = pads >> stage & 1;
    if (VEC) copies_wait<S - 1>();
    const int here = stage;
    stage = stage + 1 == S ? 0 : stage + 1;
    auto input = [&](int tensor, const void* p, int64_t ld, int i, float2 (&f)[4]) {
      Vec8<T> r;
      if (VEC)
        ring.read(here, tensor, i, r);
      else
        load8<T, VEC>(static_cast<const T*>(p) + (int64_t)row * ld, base[i], lane, D, r);
      unpack(r, f);
    };
    auto input_dh = [&](int i, float2 (&f)[4]) {
      if (VEC || a.dh) {
        input(TENSORS - 1, a.dh, a.ld_dh, i, f);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = both(0.f);
      }
    };
    if (pad) {
      const float2 zero[4] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        store8<T, VEC>(dx, base[i], lane, D, zero);
        if (DROP) {
          float2 f[4];
          input_dh(i, f);
          store8<T, VEC>(dres, base[i], lane, D, f);
        }
      }
      continue;
    }
    float2 x[NV][4], g[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      input(0, a.x, a.ld_x, i, x[i]);
      input(1, a.dy, a.ld_dy, i, g[i]);
    }
    // columns past D are zero in x and dy
    float2 p = lane_sum<NV>([&](int i, int k, float2 c) { return add2(c, x[i][k]); });
    float2 q = lane_sum<NV>([&](int i, int k, float2 c) { return ffma2(g[i][k], wv[i][k], c); });
    float sum[2] = {p.x + p.y, q.x + q.y};
    row_sums(rg, sum);
    const float mean = sum[0] * inv_d, mean_g = sum[1] * inv_d;
    p = lane_sum<NV>([&](int i, int k, float2 c) {
      x[i][k] = add2(x[i][k], inside<T, VEC>(-mean, base[i], lane, k, D));
      return ffma2(x[i][k], x[i][k], c);
    });
    q = lane_sum<NV>([&](int i, int k, float2 c) { return ffma2(mul2(g[i][k], wv[i][k]), x[i][k], c); });
    sum[0] = p.x + p.y;
    sum[1] = q.x + q.y;
    row_sums(rg, sum);
    const float rstd = rsqrtf(fmaf(sum[0], inv_d, a.eps));
    // rstd^3 alone would leave the range at spreads of 4e12 (and overflow for eps below 1e-26); rstd * S2 is of g's size
    const float2 r2 = both(rstd), c1 = both(-rstd * mean_g), c2 = both(-rstd * (rstd * (rstd * (sum[1] * inv_d))));
    Kept<T, NV, VEC> kept;
    if (DROP && !a.drop_all) kept.draw(gen, (uint64_t)row * a.groups, base, lane, a.threshold << 16);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float2 o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 gr = mul2(g[i][k], r2);
        o[k] = ffma2(gr, wv[i][k], ffma2(x[i][k], c2, c1));
        dw[i][k] = ffma2(gr, x[i][k], dw[i][k]);
        db[i][k] = add2(db[i][k], g[i][k]);
      }
      if (DROP) {
        float2 f[4];
        input_dh(i, f);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = add2(o[k], f[k]);
        store8<T, VEC>(dres, base[i], lane, D, o);
        if (a.drop_all) {
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = both(0.f);
        } else {
          kept.apply(i, a.threshold << 16, o);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = mul2(o[k], both(a.factor));
      }
      store8<T, VEC>(dx, base[i], lane, D, o);
    }
  }
  float* combine = reinterpret_cast<float*>(ring_slots);       // the ring is done with
  copies_wait<0>();
  if (R > 1) __syncthreads();
  float* out = a.partials + (int64_t)blockIdx.x * 2 * D;
  for (int g = 0; g < R; ++g) {
    if (group == g) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int c = column<T, VEC>(base[i], lane, k);
          if (c >= D) continue;
          float sw = k & 1 ? dw[i][k / 2].y : dw[i][k / 2].x, sb = k & 1 ? db[i][k / 2].y : db[i][k / 2].x;
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
    if (g + 1 < R) __syncthreads();
  }
}

// dw and db: the sums over the CTAs' partial rows, in a fixed order.  32 columns a CTA, 32 warps striding the rows.
template <typename T>
__global__ void __launch_bounds__(1024) ln_param_grad_kernel(const float* __restrict__ partials, int rows, int D,
                                                             void* dweight, void* dbias, int fp32) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;            // column of [dw | db]
  kernel_wait_ahead();
  float s = 0.f;
  if (c < 2 * D)
    for (int r = warp; r < rows; r += 32) s += __ldcg(partials + (int64_t)r * 2 * D + c);
  part[warp][lane] = s;
  __syncthreads();
  s = part[lane][warp];                            // warp w adds column w
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int k = blockIdx.x * 32 + warp;
  if (lane == 0 && k < 2 * D) {
    void* dst = k < D ? dweight : dbias;
    const int at = k < D ? k : k - D;
    if (fp32)
      static_cast<float*>(dst)[at] = s;
    else
      static_cast<T*>(dst)[at] = from_f32<T>(s);
  }
}

// out = residual + dropout(x): a thread takes four groups of eight columns, so that their loads are under way
// together.  FLAT (dense 16-byte aligned tensors without lengths): group g lies at element 8 g.  `n` groups from row
// `row0` on, fewer than 2^31.
constexpr int kDropUnroll = 4;

template <typename T, bool VEC, bool FLAT, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(RowArgs a, int64_t row0, uint32_t n) {
  const int D = a.D;
  const int64_t group0 = row0 * a.groups;
  const uint32_t block0 = blockIdx.x * (256u * kDropUnroll) + threadIdx.x;
  Vec8<T> xq[kDropUnroll], rq[kDropUnroll];
  bool there[kDropUnroll], use[kDropUnroll];
  int64_t row[kDropUnroll] = {};
  int col[kDropUnroll] = {};
  auto get = [&](const void* p, int64_t ld, int u, Vec8<T>& q) {
    if (VEC) {
      const T* src = static_cast<const T*>(p) + (FLAT ? (group0 + block0 + u * 256u) * 8 : row[u] * ld + col[u]);
#pragma unroll
      for (int i = 0; i < Vec8<T>::Q; ++i) q.q[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
    } else {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = col[u] + k < D ? to_f32(static_cast<const T*>(p)[row[u] * ld + col[u] + k]) : 0.f;
      pack(f, q);
    }
  };
#pragma unroll
  for (int u = 0; u < kDropUnroll; ++u) {
    const uint32_t g = block0 + u * 256u;
    there[u] = g < n;
    use[u] = there[u] && !a.drop_all;
    if (!FLAT && there[u]) {
      const uint32_t r = g / (uint32_t)a.groups;
      row[u] = row0 + r;
      col[u] = (int)(g - r * (uint32_t)a.groups) * 8;
      use[u] = use[u] && !padding_row(a, (uint32_t)row[u]);
    }
    if (use[u]) get(a.x, a.ld_x, u, xq[u]);
    if (RES && there[u]) get(a.residual, a.ld_res, u, rq[u]);
  }
  const Generator gen = load_generator(a.rng, a.site);
  uint64_t groups[kDropUnroll];
  uint4 drawn[kDropUnroll];
#pragma unroll
  for (int u = 0; u < kDropUnroll; ++u) groups[u] = group0 + block0 + u * 256u;
  philox(gen, groups, drawn);
#pragma unroll
  for (int u = 0; u < kDropUnroll; ++u) {
    if (!there[u]) continue;
    const uint64_t group = groups[u];
    float2 v[4] = {};
    if (RES) unpack(rq[u], v);
    if (use[u]) {
      float2 f[4];
      unpack(xq[u], f);
      keep8(drawn[u], a.threshold << 16, f);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = RES ? ffma2(f[k], both(a.factor), v[k]) : mul2(f[k], both(a.factor));
    }
    T* dst = static_cast<T*>(a.y) + (FLAT ? (int64_t)group * 8 : row[u] * D + col[u]);
    if (VEC) {
      Vec8<T> q;
      pack(v, q);
#pragma unroll
      for (int i = 0; i < Vec8<T>::Q; ++i) *(reinterpret_cast<uint4*>(dst) + i) = q.q[i];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col[u] + k < D) dst[k] = from_f32<T>(k & 1 ? v[k / 2].y : v[k / 2].x);
    }
  }
}

// The same off the 16-byte grid: a warp takes a block of 256 columns of a row, so that its single elements stay
// neighbours (eight of a lane's own in a row write every 32-byte sector eight times).
template <typename T>
__global__ void __launch_bounds__(256) dropout_block_kernel(RowArgs a) {
  const int lane = threadIdx.x & 31, D = a.D;
  const uint32_t blocks = (uint32_t)(D + 255) / 256;
  const int64_t n = a.M * blocks, step = (int64_t)gridDim.x * 8;
  const Generator gen = load_generator(a.rng, a.site);
  for (int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); item < n; item += step) {
    const int64_t row = blocks == 1 ? item : item / blocks;
    const int base[1] = {(int)(item - row * blocks) * 256};
    const bool use = !a.drop_all && !padding_row(a, (uint32_t)row);
    Vec8<T> xq, rq;
    if (use) load8<T, false>(static_cast<const T*>(a.x) + row * a.ld_x, base[0], lane, D, xq);
    if (a.residual) load8<T, false>(static_cast<const T*>(a.residual) + row * a.ld_res, base[0], lane, D, rq);
    float2 v[4] = {};
    if (a.residual) unpack(rq, v);
    if (use) {
      Kept<T, 1, false> kept;
      kept.draw(gen, (uint64_t)row * a.groups, base, lane, a.threshold << 16);
      float2 f[4];
      unpack(xq, f);
      kept.apply(0, 0, f);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = ffma2(f[k], both(a.factor), v[k]);
    }
    store8<T, false>(static_cast<T*>(a.y) + row * D, base[0], lane, D, v);
  }
}

// A row's warps and blocks of 256 columns a warp.  Two blocks, 16 columns a lane, leave 16 warps an SM beside the
// weights and the sums of their gradients in registers; the widest rows take four.  At 73728 x 1024 bf16 backward, fused
// with dropout, two blocks take 123 us and four 122, one block 158; of the odd 11376 x 1001, 36, 51 and 32 us.  One shape
// a width: the partial rows of the weights' gradients are counted before anything is known of the rows' alignment.
struct RowShape {
  int W, NV, warps;
};
RowShape row_shape(int D) {
  const int blocks = (D + 255) / 256;
  RowShape s{1, blocks == 1 ? 1 : 2, 8};
  while (s.W < 8 && s.W * s.NV < blocks) s.W *= 2;
  if (s.W * s.NV < blocks) s.NV = 4;
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

constexpr size_t kMostSums = (size_t)2 * (kMaxRowWidth / 2) * sizeof(float);     // R > 1: half the widest row

template <typename T, int NV, bool VEC, bool DROP>
int launch_fwd(const RowArgs& a, const RowShape& s, cudaStream_t stream) {
  const int R = s.warps / s.W;
  const int64_t want = (a.M + R - 1) / R, most = 2 * device_sm_count();
  constexpr int words = Ring<T, NV, DROP ? 2 : 1>::WORDS;
  const size_t smem = VEC ? sizeof(uint4) * ring_stages(words) * words * kRowThreads : 0;
  auto* kernel = ln_fwd_kernel<T, NV, VEC, DROP>;
  static std::atomic<uint64_t> allowed{0};         // an instantiation's ring is fixed, its sums are 32 KB at most
  if (smem > 32 * 1024)                            // with the static part, more than a launch gets unasked
    if (int rc = allow_smem((const void*)kernel, smem > kMostSums ? smem : kMostSums, allowed)) return rc;
  kernel<<<(int)(want < most ? want : most), kRowThreads, smem, stream>>>(a);
  return (int)cudaGetLastError();
}

template <typename T, int NV, bool VEC, bool DROP>
int launch_bwd(const RowArgs& a, const RowShape& s, cudaStream_t stream) {
  const int R = s.warps / s.W;
  constexpr int words = Ring<T, NV, DROP ? 3 : 2>::WORDS;
  const size_t ring = VEC ? sizeof(uint4) * ring_stages(words) * words * kRowThreads : 0;
  const size_t sums = R > 1 ? (size_t)2 * a.D * sizeof(float) : 0, smem = std::max(ring, sums);
  auto* kernel = ln_bwd_kernel<T, NV, VEC, DROP>;
  static std::atomic<uint64_t> allowed{0};         // an instantiation's ring is fixed, its sums are 32 KB at most
  if (smem > 32 * 1024)                            // with the static part, more than a launch gets unasked
    if (int rc = allow_smem((const void*)kernel, smem > kMostSums ? smem : kMostSums, allowed)) return rc;
  kernel<<<(int)a.partial_rows, kRowThreads, smem, stream>>>(a);
  return (int)cudaGetLastError();
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

template <typename T, bool RES>
int launch_dropout(const RowArgs& a, bool vec, cudaStream_t stream) {
  const bool flat = vec && !a.lengths && (a.ld_x == a.D || a.M == 1) && (!RES || a.ld_res == a.D || a.M == 1);
  // Blocks where they are at least 11 twentieths full.  30 M elements of bf16 without a residual: 55 us at D = 1001, 80
  // us at 150, 84 at 141, 86 at 137, 90 at 131, 96 at 121, 115 at 100; eight neighbours a lane 90 to 92 us at each.
  const int64_t blocks = (a.D + 255) / 256;
  if (!vec && (int64_t)a.D * 20 >= blocks * 256 * 11) {
    const int64_t want = (a.M * blocks + 7) / 8, most = 8 * device_sm_count();
    dropout_block_kernel<T><<<(int)(want < most ? want : most), 256, 0, stream>>>(a);
    return (int)cudaGetLastError();
  }
  const int64_t rows_a_time = (int64_t)0x7fffffff / a.groups;    // whole rows, a 32-bit count of groups a launch
  for (int64_t row0 = 0; row0 < a.M; row0 += rows_a_time) {
    const int64_t rows = a.M - row0 < rows_a_time ? a.M - row0 : rows_a_time;
    const uint32_t n = (uint32_t)(rows * a.groups);
    const int grid = (int)((n + 256u * kDropUnroll - 1) / (256u * kDropUnroll));
    if (flat)
      dropout_kernel<T, true, true, RES><<<grid, 256, 0, stream>>>(a, row0, n);
    else if (vec)
      dropout_kernel<T, true, false, RES><<<grid, 256, 0, stream>>>(a, row0, n);
    else
      dropout_kernel<T, false, false, RES><<<grid, 256, 0, stream>>>(a, row0, n);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
  }
  return 0;
}

template <typename T>
int launch_typed(RowArgs a, int op, cudaStream_t stream) {
  const bool vec = vec_ok(a, sizeof(T));
  if (a.lengths && a.M > 0) {                      // row / T = (umulhi(factor, row) + row) >> shift
    while (((uint64_t)1 << a.div_shift) < (uint64_t)a.T) ++a.div_shift;
    a.div_factor = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << a.div_shift) - a.T)) / a.T + 1);
  }
  if (op == kRowDropout) return a.residual ? launch_dropout<T, true>(a, vec, stream) : launch_dropout<T, false>(a, vec, stream);
  const bool drop = op == kRowDropNorm || op == kRowDropNormGrad, bwd = op == kRowNormGrad || op == kRowDropNormGrad;
  if (a.M > 0) {
    const int rc = drop ? (vec ? launch_rows<T, true, true>(a, bwd, stream) : launch_rows<T, false, true>(a, bwd, stream))
                        : (vec ? launch_rows<T, true, false>(a, bwd, stream)
                               : launch_rows<T, false, false>(a, bwd, stream));
    if (rc) return rc;
  }
  if (bwd) {
    return launch_behind(ln_param_grad_kernel<T>, dim3((2 * a.D + 31) / 32), 1024, 0, stream, a.partials,
                         (int)a.partial_rows, a.D, a.dweight, a.dbias, a.param_fp32);     // zeros where there are no rows
  }
  return 0;
}

}  // namespace rows_impl

// CTAs of the backward pass, a partial row each: as many as are resident
int row_partial_rows(int64_t M, int D) {
  const rows_impl::RowShape s = rows_impl::row_shape(D);
  const int R = s.warps / s.W;
  const int64_t want = (M + R - 1) / R, most = (s.NV < 4 ? 2 : 1) * device_sm_count();
  return (int)(want < most ? want : most);
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
