// Norm of queries and keys per head and rotation by the token's position, in one pass over packed tokens q | k | v:
//   x^ = x / sqrt(mean x^2 + eps),   y = x^ * w,   pairs (y_a, y_b) of the first R values of a head turned by theta_j,
//   theta_j = position_{axis(j)} * inv_freq_j;  v is copied.
// Backward:  g = the turn undone on dy,   dx = rstd (w g - x^ mean(w g x^)),   dw = sum over tokens and heads of g x^.
// The library route is a dozen passes over fp32 copies of the tokens; both directions here are bound by memory: every value is read
// once and written once.
//
// A warp takes a token (or, when tokens are few, some heads of one).  First its lanes compute one angle each - once per token, shared by
// all heads - then groups of lanes take a head each, eight values per lane.  Angles are formed and reduced to a turn in 64 bits, so that
// far positions (seconds, not only places in a sequence) keep full accuracy; sine and cosine of the remainder are fp32.  A rotation and
// its scale are two factors per value (A x + B x_partner), so that a head costs little more than its loads; the partner values come
// from L1.  Statistics and sums are fp32, one rounding at the end.
// dw is summed in registers over a warp's tokens, then over the block and by a second kernel over the blocks, in a fixed order.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

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
  int split;    // warps per token
  int lp_log2;  // lanes of a head: power of two >= Dh / 8
  float* dw_part;  // backward: [blocks, 2, Dh]
};

template <typename T>
__device__ __forceinline__ void rot_load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void rot_load8<float>(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <>
__device__ __forceinline__ void rot_load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = __uint_as_float(u[k] << 16);
    v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void rot_load8<__half>(const __half* p, float (&v)[8]) {
  const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
    v[2 * k] = f.x;
    v[2 * k + 1] = f.y;
  }
}

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

// c[k], s[k]: factors of the lane's values d0..d0+7 and of their partners (sign of the forward turn included)
template <int PAIRS>
__device__ __forceinline__ void rot_factors(const float2* cs, int d0, int n_freq, float (&c)[8], float (&s)[8]) {
  const int R = 2 * n_freq;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int d = d0 + k;
    const bool in = d < R;
    int j;
    bool first;
    if constexpr (PAIRS == ROT_NEIGHBOURS) {
      j = d >> 1;
      first = (k & 1) == 0;
    } else {
      first = d < n_freq;
      j = first ? d : d - n_freq;
    }
    const float2 f = in ? cs[j] : make_float2(1.f, 0.f);
    c[k] = f.x;
    s[k] = first ? -f.y : f.y;
  }
}

template <typename T, int PAIRS>
__device__ __forceinline__ void rot_partner(const T* head, int d0, int n_freq, const float (&x)[8], float (&xp)[8]) {
  if constexpr (PAIRS == ROT_NEIGHBOURS) {
#pragma unroll
    for (int k = 0; k < 8; ++k) xp[k] = x[k ^ 1];
  } else if constexpr (PAIRS == ROT_HALVES) {
    const int p = d0 < n_freq ? d0 + n_freq : (d0 < 2 * n_freq ? d0 - n_freq : d0);
    rot_load8(head + p, xp);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = d0 + k, p = d < n_freq ? d + n_freq : (d < 2 * n_freq ? d - n_freq : d);
      xp[k] = rot_load1(head + p);
    }
  }
}

template <int PAIRS>
__device__ __forceinline__ void rot_partner_weight(const float* w, int d0, int n_freq, float (&wp)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int d = d0 + k;
    const int p = PAIRS == ROT_NEIGHBOURS ? d ^ 1 : (d < n_freq ? d + n_freq : (d < 2 * n_freq ? d - n_freq : d));
    wp[k] = w[p];
  }
}

// sum over the lanes of a head (its power-of-two group of lanes)
__device__ __forceinline__ float rot_group_sum(float v, int lp_log2) {
  for (int o = 1 << lp_log2 >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int PAIRS, bool BWD>
__global__ void __launch_bounds__(kRotThreads) qk_norm_rotary_kernel(const RotaryParams p) {
  __shared__ __align__(16) float2 cs_all[kRotWarps][kRotMaxDim / 2];
  __shared__ __align__(16) float w_s[2][kRotMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float2* cs = cs_all[warp];
  for (int d = threadIdx.x; d < p.Dh; d += kRotThreads) {
    w_s[0][d] = p.qw ? p.qw[d] : 1.f;
    w_s[1][d] = p.kw ? p.kw[d] : 1.f;
  }
  // this lane's frequencies in turns, and the axis whose position each takes
  double freq[4];
  int axis[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = lane + 32 * i;
    freq[i] = j < p.n_freq ? p.inv_freq[j] * 0.15915494309189533577 : 0.0;
    int a = 0;
    while (a < p.axes - 1 && j >= p.axis_end[a]) ++a;
    axis[i] = a;
  }
  __syncthreads();
  const int lp = 1 << p.lp_log2, group = lane >> p.lp_log2, li = lane & (lp - 1), d0 = li * 8;
  const bool in_head = d0 < p.Dh;
  const int per_pass = 32 >> p.lp_log2, heads = p.Hq + 2 * p.Hk, turned = p.Hq + p.Hk, passes = (heads + per_pass - 1) / per_pass;
  const float inv_dim = 1.f / float(p.Dh);
  float dwq[8], dwk[8];
  if constexpr (BWD) {
#pragma unroll
    for (int k = 0; k < 8; ++k) dwq[k] = dwk[k] = 0.f;
  }
  const int64_t items = p.T * p.split, step = int64_t(gridDim.x) * kRotWarps;
  for (int64_t item = int64_t(blockIdx.x) * kRotWarps + warp; item < items; item += step) {
    const int64_t token = p.split == 1 ? item : item / p.split;
    const int part = p.split == 1 ? 0 : int(item - token * p.split);
    __syncwarp();  // the previous token's angles have been read
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = lane + 32 * i;
      if (j < p.n_freq) {
        const int64_t at = axis[i] * p.pos_axis + token * p.pos_token;
        const double pos = p.pos64 ? double(reinterpret_cast<const int64_t*>(p.positions)[at]) : double(reinterpret_cast<const int*>(p.positions)[at]);
        double turn = pos * freq[i];
        turn -= rint(turn);
        float s, c;
        sincospif(2.f * float(turn), &s, &c);
        cs[j] = make_float2(c, s);
      }
    }
    __syncwarp();
    const T* row = reinterpret_cast<const T*>(p.qkv) + token * p.ld;
    T* out = reinterpret_cast<T*>(p.out) + token * heads * p.Dh;
    const T* drow = BWD ? reinterpret_cast<const T*>(p.dy) + token * p.ld_dy : nullptr;
    float c[8], s[8];
    rot_factors<PAIRS>(cs, in_head ? d0 : 0, p.n_freq, c, s);
    for (int pass = part; pass < passes; pass += p.split) {
      const int head = pass * per_pass + group;
      const bool here = in_head && head < heads;
      const int off = head * p.Dh;
      if (here && head >= turned) {  // v
        float v[8];
        rot_load8((BWD ? drow : row) + off + d0, v);
        rot_store8(out + off + d0, v);
      }
      const bool act = here && head < turned;
      if (!__any_sync(0xffffffffu, act)) continue;
      const float* w = w_s[head < p.Hq ? 0 : 1];
      float x[8];
      if (act) {
        rot_load8(row + off + d0, x);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = 0.f;
      }
      if constexpr (!BWD) {
        float xp[8], wp[8];
        if (act) rot_partner<T, PAIRS>(row + off, d0, p.n_freq, x, xp);
        float sq = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) sq += x[k] * x[k];
        sq = rot_group_sum(sq, p.lp_log2);
        if (act) {
          const float rstd = p.norm ? 1.f / sqrtf(sq * inv_dim + p.eps) : 1.f;
          rot_partner_weight<PAIRS>(w, d0, p.n_freq, wp);
          float y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = rstd * (c[k] * w[d0 + k] * x[k] + s[k] * wp[k] * xp[k]);
          rot_store8(out + off + d0, y);
        }
      } else {
        float g[8], gp[8];
        float sq = 0.f, dot = 0.f;
        if (act) {
          rot_load8(drow + off + d0, g);
          rot_partner<T, PAIRS>(drow + off, d0, p.n_freq, g, gp);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            g[k] = c[k] * g[k] - s[k] * gp[k];
            sq += x[k] * x[k];
            dot += w[d0 + k] * g[k] * x[k];
          }
        }
        sq = rot_group_sum(sq, p.lp_log2);
        dot = rot_group_sum(dot, p.lp_log2);
        if (act) {
          const float rstd = p.norm ? 1.f / sqrtf(sq * inv_dim + p.eps) : 1.f;
          const float back = p.norm ? rstd * rstd * dot * inv_dim : 0.f;
          float dx[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) dx[k] = rstd * (w[d0 + k] * g[k] - x[k] * back);
          rot_store8(out + off + d0, dx);
          if (p.dw_part != nullptr) {
            const bool q = head < p.Hq;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float v = g[k] * x[k] * rstd;
              dwq[k] += q ? v : 0.f;
              dwk[k] += q ? 0.f : v;
            }
          }
        }
      }
    }
  }
  if constexpr (BWD) {
    if (p.dw_part == nullptr) return;
    // over the groups of the warp, then over the warps of the block, in a fixed order
    float* red = reinterpret_cast<float*>(cs_all);  // [warps][Dh]: the angles are done with
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float v = which ? dwk[k] : dwq[k];
        for (int o = lp; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (group == 0 && in_head) red[warp * kRotMaxDim + d0 + k] = v;
      }
      __syncthreads();
      for (int d = threadIdx.x; d < p.Dh; d += kRotThreads) {
        float v = 0.f;
        for (int q = 0; q < kRotWarps; ++q) v += red[q * kRotMaxDim + d];
        p.dw_part[(int64_t(blockIdx.x) * 2 + which) * p.Dh + d] = v;
      }
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
  // a warp per token, or, when the tokens would not give every SM 16 warps, its heads dealt to several
  const int sms = at::cuda::getDeviceProperties(qkv.device().index())->multiProcessorCount;
  const int64_t per_pass = 32 >> p.lp_log2, passes = (Hq + 2 * Hk + per_pass - 1) / per_pass;
  p.split = int(std::max<int64_t>(1, std::min<int64_t>(passes, 16LL * sms / T)));
  const int64_t warps = T * p.split;
  const int blocks = int(std::min<int64_t>((warps + kRotWarps - 1) / kRotWarps, (bwd ? 4 : 6) * sms));
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
