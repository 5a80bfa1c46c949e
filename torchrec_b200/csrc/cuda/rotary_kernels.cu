// Norm of queries and keys per head and rotation by the token's position, in one pass over packed tokens q | k | v:
//   x^ = x / sqrt(mean x^2 + eps),   y = x^ * w,   pairs (y_a, y_b) of the first R values of a head turned by theta_j,
//   theta_j = position_{axis(j)} * inv_freq_j;  v is copied.
// Backward:  g = the turn undone on dy,   dx = rstd (w g - x^ mean(w g x^)),   dw = sum over tokens and heads of g x^.
// The library route is a dozen passes over fp32 copies of the tokens; both directions here are bound by memory: every value is read
// once and written once.
//
// A group of lanes takes a token (eight values of a head per lane) and walks its heads; when tokens are few their heads are dealt to several
// warps.  The angles are computed once per token, each by one lane, in 64 bits and reduced to a turn there, so that far positions (seconds,
// not only places in a sequence) keep full accuracy.  What is the same for all heads - factors, weights - stays in registers, so that a
// head costs its loads, one sum over the group and two products per value; the partner's values come from the neighbouring lanes.  (With a
// warp per token and the factors fetched anew for every head, the kernel issued 600 to 900 instructions per token of 12 heads and was
// bound by that.)  Statistics and sums are fp32, one rounding at the end.
// Measured (B200): 450563 tokens of 12 heads of 64 bf16 forward 253 us (5.5 TB/s of 6.5), backward 456 us (4.0 TB/s: 0.54 instructions a
// cycle at the 24 warps an SM that its registers are bounded for); 20011 tokens of 20 heads of 128 fp32 73 us (5.6 TB/s) and 114 us
// (5.3 TB/s).  Heads whose half of the rotated part is not a multiple of eight fetch their partners one by one: 2.4 TB/s (131075 tokens of
// 24 heads of 48, 24 of them turned, fp16: 252 us, backward 333 us).
// dw is summed per token in registers, over a thread's tokens in shared memory, then over the block and by a second kernel over the
// blocks, in a fixed order.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <type_traits>

#include "common.cuh"
#include "transformer_ops.h"

namespace trb {

constexpr int kRotThreads = 256;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kRotMaxDim = 256;
constexpr int kRotMaxAxes = 8;

struct RotaryParams {
  const void* qkv;
  int64_t ld;
  const void* dy;
  int64_t ld_dy;
  void* out;              // [T, heads * Dh], contiguous
  const void* positions;  // int32 or int64
  int64_t pos_axis, pos_token;
  int pos64;
  const double* inv_freq;
  int n_freq, axes;
  int axis_end[kRotMaxAxes];
  const float* qw;  // or null
  const float* kw;
  float eps;
  int norm;
  int64_t T;
  int Hq, Hk, Dh;
  int split;    // warps that share a token's heads
  int lp_log2;  // lanes of a head: power of two >= Dh / 8
  float* dw_part;  // backward: [blocks, 2, Dh]
};

// eight values as they lie in memory, loaded ahead of their use
template <typename T>
struct RotRaw {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = u; }
  __device__ __forceinline__ RotRaw from_lane(int lane) const {
    RotRaw r;
    r.u = make_uint4(__shfl_sync(0xffffffffu, u.x, lane), __shfl_sync(0xffffffffu, u.y, lane), __shfl_sync(0xffffffffu, u.z, lane), __shfl_sync(0xffffffffu, u.w, lane));
    return r;
  }
  __device__ __forceinline__ void unpack(float (&v)[8]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
      } else {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    }
  }
};
template <>
struct RotRaw<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
  __device__ __forceinline__ RotRaw from_lane(int lane) const {
    RotRaw r;
    r.a = make_float4(__shfl_sync(0xffffffffu, a.x, lane), __shfl_sync(0xffffffffu, a.y, lane), __shfl_sync(0xffffffffu, a.z, lane), __shfl_sync(0xffffffffu, a.w, lane));
    r.b = make_float4(__shfl_sync(0xffffffffu, b.x, lane), __shfl_sync(0xffffffffu, b.y, lane), __shfl_sync(0xffffffffu, b.z, lane), __shfl_sync(0xffffffffu, b.w, lane));
    return r;
  }
  __device__ __forceinline__ void unpack(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};

__device__ __forceinline__ float rot_load1(const float* p) { return __ldg(p); }
__device__ __forceinline__ float rot_load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float rot_load1(const __half* p) { return __half2float(*p); }

__device__ __forceinline__ void rot_store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void rot_store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint4 o;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
  *reinterpret_cast<uint4*>(p) = o;
}
__device__ __forceinline__ void rot_store8(__half* p, const float (&v)[8]) {
  uint4 o;
  __half2* h = reinterpret_cast<__half2*>(&o);
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
  *reinterpret_cast<uint4*>(p) = o;
}

// How the partner of a lane's eight values is found: pairs of neighbours are in the lane; pairs half the rotated part apart are eight
// consecutive values of another lane when that half is a multiple of eight, and single values otherwise.
enum RotPairs : int { ROT_NEIGHBOURS = 0, ROT_HALVES = 1, ROT_HALVES_ODD = 2 };

__device__ __forceinline__ void rot_smem8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// c[k], s[k]: factors of the lane's values d0..d0+7 and of their partners (sign of the forward turn included)
template <int PAIRS>
__device__ __forceinline__ void rot_factors(const float2* cs, int d0, int n_freq, float (&c)[8], float (&s)[8]) {
  const int R = 2 * n_freq;
  if constexpr (PAIRS == ROT_HALVES) {
    // eight consecutive angles, or none
    if (d0 < R) {
      const float4* f = reinterpret_cast<const float4*>(cs + (d0 < n_freq ? d0 : d0 - n_freq));
      const float sign = d0 < n_freq ? -1.f : 1.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 v = f[k];
        c[2 * k] = v.x;
        s[2 * k] = sign * v.y;
        c[2 * k + 1] = v.z;
        s[2 * k + 1] = sign * v.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        c[k] = 1.f;
        s[k] = 0.f;
      }
    }
  } else if constexpr (PAIRS == ROT_NEIGHBOURS) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = d0 + 2 * k < R ? cs[d0 / 2 + k] : make_float2(1.f, 0.f);
      c[2 * k] = c[2 * k + 1] = f.x;
      s[2 * k] = -f.y;
      s[2 * k + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = d0 + k;
      const float2 f = d < R ? cs[d < n_freq ? d : d - n_freq] : make_float2(1.f, 0.f);
      c[k] = f.x;
      s[k] = d < n_freq ? -f.y : f.y;
    }
  }
}

template <typename T, int PAIRS>
__device__ __forceinline__ void rot_partner(const T* head, bool act, int d0, int partner_lane, int n_freq, const RotRaw<T>& raw, const float (&x)[8], float (&xp)[8]) {
  if constexpr (PAIRS == ROT_NEIGHBOURS) {
#pragma unroll
    for (int k = 0; k < 8; ++k) xp[k] = x[k ^ 1];
  } else if constexpr (PAIRS == ROT_HALVES) {
    raw.from_lane(partner_lane).unpack(xp);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = d0 + k, p = d < n_freq ? d + n_freq : (d < 2 * n_freq ? d - n_freq : d);
      xp[k] = act ? rot_load1(head + p) : 0.f;
    }
  }
}

// weights of the lane's values and of their partners (p0: where the partners start when they are consecutive)
template <int PAIRS>
__device__ __forceinline__ void rot_weights(const float* w, int d0, int p0, int n_freq, float (&own)[8], float (&partner)[8]) {
  rot_smem8(w + d0, own);
  if constexpr (PAIRS == ROT_NEIGHBOURS) {
#pragma unroll
    for (int k = 0; k < 8; ++k) partner[k] = own[k ^ 1];
  } else if constexpr (PAIRS == ROT_HALVES) {
    rot_smem8(w + p0, partner);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = d0 + k;
      partner[k] = w[d < n_freq ? d + n_freq : (d < 2 * n_freq ? d - n_freq : d)];
    }
  }
}

// sine and cosine of `turn` turns, |turn| <= 1/2: to 2^-23 for fp32 outputs; for 16-bit ones the hardware functions, 2^-20 off, which is
// far below half a step of the output
template <typename T>
__device__ __forceinline__ float2 rot_cos_sin(float turn) {
  float s, c;
  if constexpr (sizeof(T) == 4) sincospif(2.f * turn, &s, &c);
  else __sincosf(6.283185307179586f * turn, &s, &c);
  return make_float2(c, s);
}

// Registers are bounded so that 32 warps share an SM (forward, 16-bit types), or 24 (fp32: 83 us with 32, 71 us with 24 for 20011 tokens of
// 20 heads of 128; backward: 450 us with 24, 500 us with 16 and 524 us with 32 for 450563 tokens of 12 heads of 64).
template <typename T, bool BWD>
constexpr int kRotBlocks = BWD || sizeof(T) == 4 ? 3 : 4;

template <typename T, int PAIRS, bool BWD>
__global__ void __launch_bounds__(kRotThreads, kRotBlocks<T, BWD>) qk_norm_rotary_kernel(const RotaryParams p) {
  constexpr int kBatch = sizeof(T) == 4 ? (BWD ? 1 : 2) : (BWD ? 2 : 4);  // heads whose loads are in flight together
  __shared__ __align__(16) float2 cs_all[kRotWarps][kRotMaxDim / 2];  // a warp's tokens x frequencies (their product is at most 128)
  __shared__ __align__(16) float w_s[2][kRotMaxDim];
  __shared__ double freq_s[kRotMaxDim / 2];   // in turns
  __shared__ int64_t axis_s[kRotMaxDim / 2];  // offset of the axis' positions
  __shared__ __align__(16) float dw_s[BWD ? 2 * kRotThreads * 8 : 4];  // [q, k][thread][8]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = threadIdx.x; d < p.Dh; d += kRotThreads) {
    w_s[0][d] = p.qw ? p.qw[d] : 1.f;
    w_s[1][d] = p.kw ? p.kw[d] : 1.f;
  }
  for (int j = threadIdx.x; j < p.n_freq; j += kRotThreads) {
    freq_s[j] = p.inv_freq[j] * 0.15915494309189533577;
    int a = 0;
    while (a < p.axes - 1 && j >= p.axis_end[a]) ++a;
    axis_s[j] = a * p.pos_axis;
  }
  if constexpr (BWD) {
#pragma unroll
    for (int k = 0; k < 16; ++k) dw_s[k * kRotThreads + threadIdx.x] = 0.f;
  }
  __syncthreads();
  const int lp = 1 << p.lp_log2, group = lane >> p.lp_log2, li = lane & (lp - 1), tokens = 32 >> p.lp_log2;
  const bool in_head = li * 8 < p.Dh;
  const int d0 = in_head ? li * 8 : 0;  // lanes behind the head's last follow the first and store nothing
  const int p0 = d0 >= 2 * p.n_freq ? d0 : (d0 < p.n_freq ? d0 + p.n_freq : d0 - p.n_freq);
  const int partner_lane = in_head ? lane + (p0 - d0) / 8 : lane;
  const int turned = p.Hq + p.Hk, heads = turned + p.Hk;
  float2* cs = cs_all[warp] + group * p.n_freq;
  const float inv_dim = 1.f / float(p.Dh);
  const int64_t blocks_of_tokens = (p.T + tokens - 1) / tokens, items = blocks_of_tokens * p.split, step = int64_t(gridDim.x) * kRotWarps;
  for (int64_t item = int64_t(blockIdx.x) * kRotWarps + warp; item < items; item += step) {
    int64_t first = item;
    int part = 0;
    if (p.split > 1) {
      first = item / p.split;
      part = int(item - first * p.split);
    }
    const int64_t token = first * tokens + group;
    const bool act = token < p.T && in_head;
    const int64_t safe = min(token, p.T - 1);  // lane groups behind the last token follow it and store nothing
    const T* row = reinterpret_cast<const T*>(p.qkv) + safe * p.ld;
    const T* drow = BWD ? reinterpret_cast<const T*>(p.dy) + safe * p.ld_dy : nullptr;
    T* out = reinterpret_cast<T*>(p.out) + safe * heads * p.Dh + d0;
    RotRaw<T> rx[kBatch], rg[BWD ? kBatch : 1];
    auto load = [&](int head, int end) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (head + i * p.split < end) {
          const int off = (head + i * p.split) * p.Dh + d0;
          rx[i].load(row + off);
          if constexpr (BWD) rg[i].load(drow + off);
        }
    };
    load(part, p.Hq);  // on its way while the angles are computed
    __syncwarp();      // the previous tokens' angles have been read
    for (int j = li; j < p.n_freq; j += lp) {
      const int64_t at = axis_s[j] + safe * p.pos_token;
      double turn = (p.pos64 ? double(reinterpret_cast<const int64_t*>(p.positions)[at]) : double(reinterpret_cast<const int*>(p.positions)[at])) * freq_s[j];
      turn -= rint(turn);
      cs[j] = rot_cos_sin<T>(float(turn));
    }
    __syncwarp();
    int head = part, end = p.Hq;
#pragma unroll 1
    for (int type = 0; type < 2; ++type) {  // queries, keys
      float c[8], s[8], w[8], wp[8], acc[8];
      rot_factors<PAIRS>(cs, d0, p.n_freq, c, s);
      rot_weights<PAIRS>(w_s[type], d0, p0, p.n_freq, w, wp);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if constexpr (BWD) {
          acc[k] = 0.f;
        } else {
          c[k] *= w[k];
          s[k] *= wp[k];
        }
      }
      if (type == 1) {
        end = turned;
        load(head, end);
      }
#pragma unroll 1
      while (head < end) {  // the same for all lanes
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (head + i * p.split >= end) break;
          const int off = (head + i * p.split) * p.Dh;
          float x[8];
          rx[i].unpack(x);
          if constexpr (!BWD) {
            float xp[8];
            rot_partner<T, PAIRS>(row + off, true, d0, partner_lane, p.n_freq, rx[i], x, xp);
            float sq = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) sq += x[k] * x[k];
            sq = in_head ? sq : 0.f;
            for (int o = lp >> 1; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
            const float rstd = p.norm ? rsqrtf(sq * inv_dim + p.eps) : 1.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = rstd * (c[k] * x[k] + s[k] * xp[k]);
            if (act) rot_store8(out + off, x);
          } else {
            float g[8], gp[8];
            rg[i].unpack(g);
            rot_partner<T, PAIRS>(drow + off, true, d0, partner_lane, p.n_freq, rg[i], g, gp);
            float sq = 0.f, dot = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              g[k] = c[k] * g[k] - s[k] * gp[k];
              sq += x[k] * x[k];
              gp[k] = g[k] * x[k];
              dot += w[k] * gp[k];
            }
            sq = in_head ? sq : 0.f;
            dot = in_head ? dot : 0.f;
            for (int o = lp >> 1; o > 0; o >>= 1) {
              sq += __shfl_xor_sync(0xffffffffu, sq, o);
              dot += __shfl_xor_sync(0xffffffffu, dot, o);
            }
            const float rstd = p.norm ? rsqrtf(sq * inv_dim + p.eps) : 1.f;
            const float back = p.norm ? rstd * rstd * dot * inv_dim : 0.f;
            if (act) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                acc[k] += gp[k] * rstd;
                x[k] = rstd * (w[k] * g[k] - x[k] * back);
              }
              rot_store8(out + off, x);
            }
          }
        }
        head += kBatch * p.split;
        if (head < end) load(head, end);
      }
      // the first of this warp's heads of the next type
      head = type == 0 ? part + (p.Hq - part + p.split - 1) / p.split * p.split : head;
      if constexpr (BWD) {
        if (p.dw_part != nullptr) {
          float* d = dw_s + (type * kRotThreads + threadIdx.x) * 8;
          float v[8];
          rot_smem8(d, v);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] += acc[k];
          rot_store8(d, v);
        }
      }
    }
    // v
    const T* vrow = BWD ? drow : row;
#pragma unroll 1
    for (head = part + (turned - part + p.split - 1) / p.split * p.split; head < heads; head += kBatch * p.split) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (head + i * p.split < heads) rx[i].load(vrow + (head + i * p.split) * p.Dh + d0);
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (act && head + i * p.split < heads) rx[i].store(out + (head + i * p.split) * p.Dh);
    }
  }
  if constexpr (BWD) {
    if (p.dw_part == nullptr) return;
    // over the block's threads that hold the same eight columns, in a fixed order
    __syncthreads();
    for (int d = threadIdx.x; d < 2 * p.Dh; d += kRotThreads) {
      const int which = d >= p.Dh ? 1 : 0, col = d - which * p.Dh;
      float v = 0.f;
      for (int t = col / 8; t < kRotThreads; t += lp) v += dw_s[(which * kRotThreads + t) * 8 + (col & 7)];
      p.dw_part[int64_t(blockIdx.x) * 2 * p.Dh + d] = v;
    }
  }
}

// dw [2, Dh]: one block per eight columns, 32 threads a column, in a fixed order
__global__ void __launch_bounds__(kRotThreads) qk_norm_dw_kernel(const float* __restrict__ part, int blocks, int n, float* __restrict__ dw) {
  const int lane = threadIdx.x & 31, col = blockIdx.x * kRotWarps + (threadIdx.x >> 5);
  if (col >= n) return;
  float v = 0.f;
  for (int b = lane; b < blocks; b += 32) v += part[int64_t(b) * n + col];
  v = warp_sum(v);
  if (lane == 0) dw[col] = v;
}

template <typename T, bool BWD>
static void rot_launch(const RotaryParams& p, int pairs, int blocks) {
  auto stream = at::cuda::getCurrentCUDAStream();
  if (pairs == ROT_NEIGHBOURS) qk_norm_rotary_kernel<T, ROT_NEIGHBOURS, BWD><<<blocks, kRotThreads, 0, stream>>>(p);
  else if (pairs == ROT_HALVES) qk_norm_rotary_kernel<T, ROT_HALVES, BWD><<<blocks, kRotThreads, 0, stream>>>(p);
  else qk_norm_rotary_kernel<T, ROT_HALVES_ODD, BWD><<<blocks, kRotThreads, 0, stream>>>(p);
  TRB_CUDA_CHECK(cudaGetLastError());
}

static void rot_check_rows(const at::Tensor& t, const char* name, int64_t cols) {
  const int64_t per16 = 16 / t.element_size();
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && t.size(1) == cols && t.stride(1) == 1 && t.stride(0) % per16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                  (t.size(0) <= 1 || t.stride(0) >= cols),
              "qk_norm_rotary: ", name, " has rows of (heads + 2 kv_heads) * head_dim values that start on 16 bytes");
}

// dy: none for the forward.  Returns (out [T, cols], dw [2, Dh] - empty unless the backward has weights).
static std::tuple<at::Tensor, at::Tensor> rot_run(const at::Tensor& qkv, const c10::optional<at::Tensor>& dy, const at::Tensor& positions, const at::Tensor& inv_freq,
                                                  const c10::optional<at::Tensor>& qw, const c10::optional<at::Tensor>& kw, at::IntArrayRef sections, int64_t Hq, int64_t Hk,
                                                  double eps, bool norm, bool interleaved, bool want_dw) {
  TORCH_CHECK(qkv.dim() == 2 && Hq >= 1 && Hk >= 1 && Hq <= 4096 && Hk <= 4096 && qkv.size(1) % (Hq + 2 * Hk) == 0, "qk_norm_rotary: qkv is [T, (heads + 2 kv_heads) * head_dim]");
  const int64_t T = qkv.size(0), Dh = qkv.size(1) / (Hq + 2 * Hk);
  TORCH_CHECK(Dh >= 8 && Dh % 8 == 0 && Dh <= kRotMaxDim, "qk_norm_rotary: the head dimension is a multiple of 8, at most ", kRotMaxDim);
  TORCH_CHECK(qkv.scalar_type() == at::kBFloat16 || qkv.scalar_type() == at::kHalf || qkv.scalar_type() == at::kFloat, "qk_norm_rotary: bf16, fp16 or fp32");
  rot_check_rows(qkv, "qkv", qkv.size(1));
  const bool bwd = dy.has_value() && dy->defined();
  if (bwd) {
    rot_check_rows(*dy, "the gradient", qkv.size(1));
    TORCH_CHECK(dy->scalar_type() == qkv.scalar_type() && dy->size(0) == T && dy->device() == qkv.device());
  }
  TORCH_CHECK(inv_freq.device() == qkv.device() && inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1 && inv_freq.is_contiguous() && inv_freq.numel() >= 1 &&
                  2 * inv_freq.numel() <= Dh,
              "qk_norm_rotary: inv_freq holds 1 to head_dim / 2 fp64 frequencies");
  const int64_t n_freq = inv_freq.numel();
  TORCH_CHECK(positions.device() == qkv.device() && (positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt) && positions.dim() == 2 &&
                  positions.size(0) == int64_t(sections.size()) && positions.size(1) == T && positions.size(0) <= kRotMaxAxes,
              "qk_norm_rotary: positions is an integer [axes, T] with at most ", kRotMaxAxes, " axes");
  RotaryParams p{};
  int64_t end = 0;
  for (size_t a = 0; a < sections.size(); ++a) {
    TORCH_CHECK(sections[a] >= 0, "qk_norm_rotary: a section is negative");
    end += sections[a];
    p.axis_end[a] = int(end);
  }
  TORCH_CHECK(end == n_freq, "qk_norm_rotary: the sections add up to ", end, " of ", n_freq, " frequencies");
  for (const auto* w : {&qw, &kw})
    if (w->has_value() && (*w)->defined())
      TORCH_CHECK((*w)->device() == qkv.device() && (*w)->scalar_type() == at::kFloat && (*w)->dim() == 1 && (*w)->numel() == Dh && (*w)->is_contiguous(),
                  "qk_norm_rotary: a norm weight is fp32 [head_dim]");
  c10::cuda::CUDAGuard guard(qkv.device());
  at::Tensor out = at::empty({T, qkv.size(1)}, qkv.options());
  at::Tensor dw = at::empty({want_dw ? 2 : 0, Dh}, qkv.options().dtype(at::kFloat));
  if (T == 0) {
    dw.zero_();
    return {out, dw};
  }
  p.qkv = qkv.data_ptr();
  p.ld = qkv.stride(0);
  p.dy = bwd ? dy->data_ptr() : nullptr;
  p.ld_dy = bwd ? dy->stride(0) : 0;
  p.out = out.data_ptr();
  p.positions = positions.data_ptr();
  p.pos_axis = positions.stride(0);
  p.pos_token = positions.stride(1);
  p.pos64 = positions.scalar_type() == at::kLong;
  p.inv_freq = inv_freq.data_ptr<double>();
  p.n_freq = int(n_freq);
  p.axes = int(sections.size());
  p.qw = qw.has_value() && qw->defined() ? qw->data_ptr<float>() : nullptr;
  p.kw = kw.has_value() && kw->defined() ? kw->data_ptr<float>() : nullptr;
  p.eps = float(eps);
  p.norm = norm;
  p.T = T;
  p.Hq = int(Hq);
  p.Hk = int(Hk);
  p.Dh = int(Dh);
  while ((8 << p.lp_log2) < Dh) ++p.lp_log2;
  // a group of lanes per token, or, when the tokens would not give every SM 16 warps, its heads dealt to several warps
  const int sms = at::cuda::getDeviceProperties(qkv.device().index())->multiProcessorCount;
  const int64_t groups = (T + (32 >> p.lp_log2) - 1) / (32 >> p.lp_log2);
  p.split = int(std::max<int64_t>(1, std::min<int64_t>(Hq + 2 * Hk, 16LL * sms / groups)));
  const int64_t warps = groups * p.split;
  const int blocks = int(std::min<int64_t>((warps + kRotWarps - 1) / kRotWarps, (bwd || qkv.scalar_type() == at::kFloat ? 3 : 4) * sms));
  at::Tensor part;
  if (want_dw) {
    part = at::empty({blocks, 2, Dh}, dw.options());
    p.dw_part = part.data_ptr<float>();
  }
  const int pairs = interleaved ? ROT_NEIGHBOURS : (n_freq % 8 == 0 ? ROT_HALVES : ROT_HALVES_ODD);
  if (qkv.scalar_type() == at::kBFloat16) bwd ? rot_launch<__nv_bfloat16, true>(p, pairs, blocks) : rot_launch<__nv_bfloat16, false>(p, pairs, blocks);
  else if (qkv.scalar_type() == at::kHalf) bwd ? rot_launch<__half, true>(p, pairs, blocks) : rot_launch<__half, false>(p, pairs, blocks);
  else bwd ? rot_launch<float, true>(p, pairs, blocks) : rot_launch<float, false>(p, pairs, blocks);
  if (want_dw) {
    qk_norm_dw_kernel<<<unsigned((2 * Dh + kRotWarps - 1) / kRotWarps), kRotThreads, 0, at::cuda::getCurrentCUDAStream()>>>(p.dw_part, blocks, int(2 * Dh), dw.data_ptr<float>());
    TRB_CUDA_CHECK(cudaGetLastError());
  }
  return {out, dw};
}

at::Tensor qk_norm_rotary_fwd(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& inv_freq, const c10::optional<at::Tensor>& qw,
                              const c10::optional<at::Tensor>& kw, at::IntArrayRef sections, int64_t heads, int64_t kv_heads, double eps, bool norm, bool interleaved) {
  return std::get<0>(rot_run(qkv, c10::nullopt, positions, inv_freq, qw, kw, sections, heads, kv_heads, eps, norm, interleaved, false));
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rotary_bwd(const at::Tensor& dy, const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& inv_freq,
                                                      const c10::optional<at::Tensor>& qw, const c10::optional<at::Tensor>& kw, at::IntArrayRef sections, int64_t heads,
                                                      int64_t kv_heads, double eps, bool norm, bool interleaved, bool want_dw) {
  return rot_run(qkv, dy, positions, inv_freq, qw, kw, sections, heads, kv_heads, eps, norm, interleaved, want_dw);
}

}  // namespace trb

TORCH_LIBRARY_FRAGMENT(trb200, m) {
  m.def("qk_norm_rotary_fwd(Tensor qkv, Tensor positions, Tensor inv_freq, Tensor? q_weight, Tensor? k_weight, int[] sections, int heads, int kv_heads, float eps, bool norm, "
        "bool interleaved) -> Tensor");
  m.def("qk_norm_rotary_bwd(Tensor dy, Tensor qkv, Tensor positions, Tensor inv_freq, Tensor? q_weight, Tensor? k_weight, int[] sections, int heads, int kv_heads, float eps, "
        "bool norm, bool interleaved, bool want_dw) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(trb200, CUDA, m) {
  m.impl("qk_norm_rotary_fwd", &trb::qk_norm_rotary_fwd);
  m.impl("qk_norm_rotary_bwd", &trb::qk_norm_rotary_bwd);
}
