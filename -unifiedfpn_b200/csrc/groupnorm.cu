// Group norm with an activation on channels-last maps, forward and backward, for one map or
// the levels of a pyramid in one call.
//
// Over the m = pixels * Cg values of group g of image n (Cg = C / groups adjacent channels):
//   mean = sum x / m;  var = sum (x - mean)^2 / m;  rstd = 1 / sqrt(var + eps)
//   xhat = (x - mean) * rstd;  z = xhat * weight[c] + bias[c];  y = act(z)
// and backward, with dz = dy * act'(z):
//   dbias[c] = sum dz;  dweight[c] = sum dz * xhat   (over images and pixels)
//   dx = rstd * (w dz - mean_g(w dz) - xhat * mean_g(w dz xhat))
//
// All statistics and sums are fp32.  The variance never comes from a difference of raw moments:
// every thread takes the mean of a few pixels in registers, the squares about that mean, and
// merges such (count, mean, M2) triples,
//   M2_ab = M2_a + M2_b + (mean_b - mean_a)^2 n_a n_b / (n_a + n_b),
// and fp32 values are taken relative to the group's first value of the image (the pivot), so that
// the means in between are not rounded at the height of a mean far above the spread.  (16-bit
// values have at most 11 bits: their spread is never that far below their mean.)  Every sum has a
// fixed order (no atomics): the same inputs give the same bits.
//
// The kernels move bytes: two passes over the maps (statistics, then apply), each a stream of
// 16-byte loads, the batch cut into runs of images whose maps stay in the 126 MB L2 cache, so
// that the second pass reads there instead of HBM.
#include "kernels.h"
#include "ptx.cuh"
#include "vec16.cuh"

#include <algorithm>
#include <cstring>
#include <vector>

namespace ufpn {

namespace {

constexpr int kGnThreads = 512;
constexpr int kGnBatch = 8;      // pixels per thread and step: 16-byte loads in flight
constexpr int kGnMaxRuns = 8;    // runs (images of one level) per launch
constexpr int kGnMaxChannels = 2048;  // a thread keeps one vector of a pixel: C / V <= 512

enum : int { kGnNone = 0, kGnRelu = 1, kGnLeaky = 2, kGnSwish = 3 };

// One run: consecutive images of one level, each cut into `chunks` runs of `per` pixels.
struct GnRun {
  const void* x;
  const void* g;  // backward: grad_output
  void* y;        // forward: output; backward: grad_input (null: none)
  const float* w;  // [C] or null (1)
  const float* b;  // [C] or null (0)
  float* mean;     // [N][groups]: written forward (null: not wanted), read backward
  float* rstd;
  long long pixels;  // of one image
  long long per;
  int n0, chunks;
  int first_block;  // block of image n0, chunk 0
  int row0;         // its row of partial results; a run's rows are [image][chunk]
};
struct GnArgs {
  GnRun run[kGnMaxRuns];
  int runs;
  int C, groups, cg;
  int act;
  float alpha, eps;
  float2* part;   // [row][groups]: (mean, M2) forward, (sum w dz, sum w dz xhat) backward
  float* part_c;  // backward: [row][2][C]: sum dz, sum dz xhat
  float* pivot;   // fp32 forward: [row of chunk 0][groups]
};
template <typename T>
constexpr bool kGnPivot = sizeof(T) == 4;

// exp and the division of the sigmoid: the fast forms (relative error about 2^-21) for 16-bit
// maps, whose results are rounded to 2^-9 or 2^-12 anyway; the accurate ones for fp32.
template <typename T>
__device__ __forceinline__ float gn_sigmoid(float z) {
  if constexpr (sizeof(T) == 2)
    return __fdividef(1.f, 1.f + __expf(-z));
  else
    return 1.f / (1.f + expf(-z));
}
template <typename T>
__device__ __forceinline__ float gn_act(float z, int act, float alpha) {
  if (act == kGnRelu) return fmaxf(z, 0.f);
  if (act == kGnLeaky) return z > 0.f ? z : alpha * z;
  if (act == kGnSwish) return z * gn_sigmoid<T>(z);
  return z;
}
template <typename T>
__device__ __forceinline__ float gn_act_grad(float z, int act, float alpha) {
  if (act == kGnRelu) return z > 0.f ? 1.f : 0.f;
  if (act == kGnLeaky) return z > 0.f ? 1.f : alpha;
  if (act == kGnSwish) {
    const float q = gn_sigmoid<T>(z);
    return q * fmaf(z, 1.f - q, 1.f);
  }
  return 1.f;
}
// z from x in the one form that the forward and the backward share, each step rounded on its
// own, so that both take the same side of an activation's kink.
__device__ __forceinline__ float gn_xhat(float x, float mean, float rstd) {
  return __fmul_rn(__fsub_rn(x, mean), rstd);
}

// Which run, image, chunk and pixel range this block has.
struct GnPlace {
  int run, n, chunk;
  long long p0, p1;
};
__device__ __forceinline__ GnPlace gn_place(const GnArgs& a) {
  GnPlace p;
  p.run = 0;
  while (p.run + 1 < a.runs && static_cast<int>(blockIdx.x) >= a.run[p.run + 1].first_block) ++p.run;
  const GnRun& r = a.run[p.run];
  const int b = static_cast<int>(blockIdx.x) - r.first_block;
  const int i = b / r.chunks;
  p.chunk = b - i * r.chunks;
  p.n = r.n0 + i;
  p.p0 = p.chunk * r.per;
  p.p1 = min(r.pixels, p.p0 + r.per);
  return p;
}

__device__ __forceinline__ float gn_group_sum(float v, int tpg) {
  for (int o = tpg >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Threads per group in a block's final sums over shared memory: a power of two up to a warp.
__device__ __forceinline__ int gn_threads_per_group(int groups) {
  int t = 32;
  while (t > 1 && t * groups > kGnThreads) t >>= 1;
  return t;
}

// Statistics of each block's pixels by group: part[row][g] = (mean, M2).  Thread t keeps
// channel vector t % VC and takes every PL-th pixel.
template <typename T>
__global__ void __launch_bounds__(kGnThreads, 2) gn_stats_kernel(const __grid_constant__ GnArgs a) {
  constexpr int V = Vec16<T>::V;
  __shared__ float s_mean[kGnThreads * V];  // [pixel lane][C]
  __shared__ float s_m2[kGnThreads * V];
  __shared__ float s_cnt[kGnThreads];       // [pixel lane]
  const GnPlace at = gn_place(a);
  const GnRun& r = a.run[at.run];
  const int vc = a.C / V, lanes = kGnThreads / vc;
  const int v = threadIdx.x % vc, pl = threadIdx.x / vc;
  griddep_wait();
  if (pl < lanes) {
    float mean[V], m2[V], pv[V];
    float cnt = 0.f;
    const T* x = static_cast<const T*>(r.x) + static_cast<size_t>(at.n) * r.pixels * a.C;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      mean[e] = m2[e] = 0.f;
      if constexpr (kGnPivot<T>) pv[e] = static_cast<float>(x[(v * V + e) / a.cg * a.cg]);
    }
    for (long long p = at.p0 + pl; p < at.p1; p += static_cast<long long>(lanes) * kGnBatch) {
      uint4 u[kGnBatch];
      int k_n = 0;
#pragma unroll
      for (int k = 0; k < kGnBatch; ++k) {
        const long long q = p + static_cast<long long>(k) * lanes;
        u[k] = make_uint4(0u, 0u, 0u, 0u);
        if (q < at.p1) {
          u[k] = *(reinterpret_cast<const uint4*>(x + q * a.C) + v);
          ++k_n;
        }
      }
      // mean and squares of the k_n pixels (the zeros of missing ones add nothing to the sum and
      // are left out of the squares), then one merge
      float s[V], q2[V];
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] = q2[e] = 0.f;
#pragma unroll
      for (int k = 0; k < kGnBatch; ++k) {
        float f[V];
        Vec16<T>::unpack(u[k], f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if constexpr (kGnPivot<T>)
            s[e] += k < k_n ? f[e] - pv[e] : 0.f;
          else
            s[e] += f[e];
        }
      }
      const float nb = static_cast<float>(k_n), inv = 1.f / nb;
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] *= inv;
#pragma unroll
      for (int k = 0; k < kGnBatch; ++k) {
        if (k < k_n) {
          float f[V];
          Vec16<T>::unpack(u[k], f);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float d = f[e];
            if constexpr (kGnPivot<T>) d -= pv[e];
            d -= s[e];
            q2[e] = fmaf(d, d, q2[e]);
          }
        }
      }
      const float w = nb / (cnt + nb), wn = w * cnt;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = s[e] - mean[e];
        mean[e] = fmaf(d, w, mean[e]);
        m2[e] += fmaf(d * d, wn, q2[e]);
      }
      cnt += nb;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s_mean[pl * a.C + v * V + e] = mean[e];
      s_m2[pl * a.C + v * V + e] = m2[e];
    }
    if (v == 0) s_cnt[pl] = cnt;
  }
  __syncthreads();
  griddep_launch_dependents();
  // the group's channels and pixel lanes: their mean, then the squares about it
  const int tpg = gn_threads_per_group(a.groups);
  const int j = threadIdx.x % tpg;
  const float inv_total = 1.f / (static_cast<float>(at.p1 - at.p0) * static_cast<float>(a.cg));
  float2* out = a.part + static_cast<size_t>(r.row0 + (at.n - r.n0) * r.chunks + at.chunk) * a.groups;
  for (int g0 = 0; g0 < a.groups; g0 += kGnThreads / tpg) {
    const int g = g0 + threadIdx.x / tpg;
    const bool in = g < a.groups;
    const int entries = in ? lanes * a.cg : 0;
    float s = 0.f;
    for (int i = j; i < entries; i += tpg) {
      const int l = i / a.cg, c = i - l * a.cg;
      s = fmaf(s_cnt[l], s_mean[l * a.C + g * a.cg + c], s);
    }
    const float mean = gn_group_sum(s, tpg) * inv_total;
    float m2 = 0.f;
    for (int i = j; i < entries; i += tpg) {
      const int l = i / a.cg, c = i - l * a.cg;
      const float d = s_mean[l * a.C + g * a.cg + c] - mean;
      m2 += fmaf(d * d, s_cnt[l], s_m2[l * a.C + g * a.cg + c]);
    }
    m2 = gn_group_sum(m2, tpg);
    if (in && j == 0) {
      out[g] = make_float2(mean, m2);
      if constexpr (kGnPivot<T>) {
        if (at.chunk == 0)
          a.pivot[static_cast<size_t>(r.row0 + (at.n - r.n0) * r.chunks) * a.groups + g] =
              static_cast<const float*>(r.x)[static_cast<size_t>(at.n) * r.pixels * a.C + g * a.cg];
      }
    }
  }
}

// y = act(z).  Every block first merges its image's rows of partial statistics (chunk 0 also
// writes them out), then streams its pixels.
template <typename T>
__global__ void __launch_bounds__(kGnThreads, 2) gn_apply_kernel(const __grid_constant__ GnArgs a) {
  constexpr int V = Vec16<T>::V;
  __shared__ float s_mean[kGnThreads], s_m2[kGnThreads], s_cnt[kGnThreads];
  __shared__ float g_mean[kGnMaxChannels], g_rstd[kGnMaxChannels];
  const GnPlace at = gn_place(a);
  const GnRun& r = a.run[at.run];
  griddep_wait();
  griddep_launch_dependents();
  const float2* rows = a.part + static_cast<size_t>(r.row0 + (at.n - r.n0) * r.chunks) * a.groups;
  const int span = min(a.groups, kGnThreads);
  const int per_g = kGnThreads / span;  // threads per group, each over every per_g-th row
  for (int g0 = 0; g0 < a.groups; g0 += span) {
    const int g = g0 + threadIdx.x % span, j = threadIdx.x / span;
    float mean = 0.f, m2 = 0.f, cnt = 0.f;
    if (j < per_g && g < a.groups) {
      for (int i = j; i < r.chunks; i += per_g) {
        const float2 t = rows[static_cast<size_t>(i) * a.groups + g];
        const float nb = static_cast<float>(min(r.per, r.pixels - i * r.per));
        const float d = t.x - mean, w = nb / (cnt + nb);
        mean = fmaf(d, w, mean);
        m2 += fmaf(d * d, w * cnt * static_cast<float>(a.cg), t.y);
        cnt += nb;
      }
      s_mean[threadIdx.x] = mean;
      s_m2[threadIdx.x] = m2;
      s_cnt[threadIdx.x] = cnt;
    }
    __syncthreads();
    if (j == 0 && g < a.groups) {
      const float px = static_cast<float>(r.pixels);
      float s = 0.f;
      for (int i = 0; i < per_g; ++i) s = fmaf(s_cnt[i * span + threadIdx.x], s_mean[i * span + threadIdx.x], s);
      float mu = s / px;
      float q = 0.f;
      for (int i = 0; i < per_g; ++i) {
        const float d = s_mean[i * span + threadIdx.x] - mu;
        q += fmaf(d * d, s_cnt[i * span + threadIdx.x] * static_cast<float>(a.cg), s_m2[i * span + threadIdx.x]);
      }
      const float rs = 1.f / sqrtf(q / (px * static_cast<float>(a.cg)) + a.eps);
      if constexpr (kGnPivot<T>)
        mu += a.pivot[static_cast<size_t>(r.row0 + (at.n - r.n0) * r.chunks) * a.groups + g];
      g_mean[g] = mu;
      g_rstd[g] = rs;
      if (at.chunk == 0 && r.mean != nullptr) {
        r.mean[static_cast<size_t>(at.n) * a.groups + g] = mu;
        r.rstd[static_cast<size_t>(at.n) * a.groups + g] = rs;
      }
    }
    __syncthreads();
  }
  const int vc = a.C / V, lanes = kGnThreads / vc;
  const int v = threadIdx.x % vc, pl = threadIdx.x / vc;
  if (pl >= lanes) return;
  float mean[V], rstd[V], w[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = v * V + e, g = c / a.cg;
    mean[e] = g_mean[g];
    rstd[e] = g_rstd[g];
    w[e] = r.w != nullptr ? __ldg(r.w + c) : 1.f;
    b[e] = r.b != nullptr ? __ldg(r.b + c) : 0.f;
  }
  const size_t base = static_cast<size_t>(at.n) * r.pixels * a.C;
  const T* x = static_cast<const T*>(r.x) + base;
  T* y = static_cast<T*>(r.y) + base;
  constexpr int K = 4;
  for (long long p = at.p0 + pl; p < at.p1; p += static_cast<long long>(lanes) * K) {
    uint4 u[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long long q = p + static_cast<long long>(k) * lanes;
      if (q < at.p1) u[k] = *(reinterpret_cast<const uint4*>(x + q * a.C) + v);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long long q = p + static_cast<long long>(k) * lanes;
      if (q < at.p1) {
        float f[V];
        Vec16<T>::unpack(u[k], f);
#pragma unroll
        for (int e = 0; e < V; ++e)
          f[e] = gn_act<T>(__fmaf_rn(gn_xhat(f[e], mean[e], rstd[e]), w[e], b[e]), a.act, a.alpha);
        *(reinterpret_cast<uint4*>(y + q * a.C) + v) = Vec16<T>::pack(f);
      }
    }
  }
}

// Loads a thread's per-channel constants of the backward.
template <int V>
struct GnChannels {
  float mean[V], rstd[V], w[V], b[V];
  __device__ __forceinline__ void load(const GnArgs& a, const GnRun& r, int n, int v) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = v * V + e;
      const size_t g = static_cast<size_t>(n) * a.groups + c / a.cg;
      mean[e] = __ldg(r.mean + g);
      rstd[e] = __ldg(r.rstd + g);
      w[e] = r.w != nullptr ? __ldg(r.w + c) : 1.f;
      b[e] = r.b != nullptr ? __ldg(r.b + c) : 0.f;
    }
  }
};

// Backward sums of each block's pixels: by channel (part_c, for dweight / dbias) and, weighted,
// by group (part, for dx).
template <typename T>
__global__ void __launch_bounds__(kGnThreads, 1) gn_bwd_stats_kernel(const __grid_constant__ GnArgs a) {
  constexpr int V = Vec16<T>::V;
  constexpr int K = 4;
  __shared__ float s_dz[kGnThreads * V];  // [pixel lane][C], then row 0 = the block's sums
  __shared__ float s_dx[kGnThreads * V];
  const GnPlace at = gn_place(a);
  const GnRun& r = a.run[at.run];
  const int vc = a.C / V, lanes = kGnThreads / vc;
  const int v = threadIdx.x % vc, pl = threadIdx.x / vc;
  griddep_wait();
  if (pl < lanes) {
    GnChannels<V> ch;
    ch.load(a, r, at.n, v);
    float sz[V], sx[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sz[e] = sx[e] = 0.f;
    const size_t base = static_cast<size_t>(at.n) * r.pixels * a.C;
    const T* x = static_cast<const T*>(r.x) + base;
    const T* dy = static_cast<const T*>(r.g) + base;
    for (long long p = at.p0 + pl; p < at.p1; p += static_cast<long long>(lanes) * K) {
      uint4 u[K], d[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const long long q = p + static_cast<long long>(k) * lanes;
        if (q < at.p1) {
          u[k] = *(reinterpret_cast<const uint4*>(x + q * a.C) + v);
          d[k] = *(reinterpret_cast<const uint4*>(dy + q * a.C) + v);
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (p + static_cast<long long>(k) * lanes < at.p1) {
          float f[V], h[V];
          Vec16<T>::unpack(u[k], f);
          Vec16<T>::unpack(d[k], h);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float xh = gn_xhat(f[e], ch.mean[e], ch.rstd[e]);
            const float dz = h[e] * gn_act_grad<T>(__fmaf_rn(xh, ch.w[e], ch.b[e]), a.act, a.alpha);
            sz[e] += dz;
            sx[e] = fmaf(dz, xh, sx[e]);
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s_dz[pl * a.C + v * V + e] = sz[e];
      s_dx[pl * a.C + v * V + e] = sx[e];
    }
  }
  __syncthreads();
  griddep_launch_dependents();
  const size_t row = r.row0 + static_cast<size_t>(at.n - r.n0) * r.chunks + at.chunk;
  float* pc = a.part_c + row * 2 * a.C;
  for (int c = threadIdx.x; c < a.C; c += kGnThreads) {
    float z = 0.f, x = 0.f;
    for (int l = 0; l < lanes; ++l) {
      z += s_dz[l * a.C + c];
      x += s_dx[l * a.C + c];
    }
    pc[c] = z;
    pc[a.C + c] = x;
    const float w = r.w != nullptr ? __ldg(r.w + c) : 1.f;
    s_dz[c] = w * z;  // (only this thread reads and writes column c)
    s_dx[c] = w * x;
  }
  __syncthreads();
  for (int g = threadIdx.x; g < a.groups; g += kGnThreads) {
    float z = 0.f, x = 0.f;
    for (int c = 0; c < a.cg; ++c) {
      z += s_dz[g * a.cg + c];
      x += s_dx[g * a.cg + c];
    }
    a.part[row * a.groups + g] = make_float2(z, x);
  }
}

template <typename T>
__global__ void __launch_bounds__(kGnThreads, 1) gn_bwd_apply_kernel(const __grid_constant__ GnArgs a) {
  constexpr int V = Vec16<T>::V;
  constexpr int K = 4;
  __shared__ float s_z[kGnThreads], s_x[kGnThreads];
  __shared__ float g_z[kGnMaxChannels], g_x[kGnMaxChannels];
  const GnPlace at = gn_place(a);
  const GnRun& r = a.run[at.run];
  griddep_wait();
  griddep_launch_dependents();
  const float2* rows = a.part + static_cast<size_t>(r.row0 + (at.n - r.n0) * r.chunks) * a.groups;
  const int span = min(a.groups, kGnThreads);
  const int per_g = kGnThreads / span;
  const float inv_m = 1.f / (static_cast<float>(r.pixels) * static_cast<float>(a.cg));
  for (int g0 = 0; g0 < a.groups; g0 += span) {
    const int g = g0 + threadIdx.x % span, j = threadIdx.x / span;
    float z = 0.f, x = 0.f;
    if (j < per_g && g < a.groups) {
      for (int i = j; i < r.chunks; i += per_g) {
        const float2 t = rows[static_cast<size_t>(i) * a.groups + g];
        z += t.x;
        x += t.y;
      }
      s_z[threadIdx.x] = z;
      s_x[threadIdx.x] = x;
    }
    __syncthreads();
    if (j == 0 && g < a.groups) {
      z = x = 0.f;
      for (int i = 0; i < per_g; ++i) {
        z += s_z[i * span + threadIdx.x];
        x += s_x[i * span + threadIdx.x];
      }
      g_z[g] = __fmul_rn(z, inv_m);
      g_x[g] = __fmul_rn(x, inv_m);
    }
    __syncthreads();
  }
  const int vc = a.C / V, lanes = kGnThreads / vc;
  const int v = threadIdx.x % vc, pl = threadIdx.x / vc;
  if (pl >= lanes) return;
  GnChannels<V> ch;
  ch.load(a, r, at.n, v);
  float mz[V], mx[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int g = (v * V + e) / a.cg;
    mz[e] = g_z[g];
    mx[e] = g_x[g];
  }
  const size_t base = static_cast<size_t>(at.n) * r.pixels * a.C;
  const T* x = static_cast<const T*>(r.x) + base;
  const T* dy = static_cast<const T*>(r.g) + base;
  T* dx = static_cast<T*>(r.y) + base;
  for (long long p = at.p0 + pl; p < at.p1; p += static_cast<long long>(lanes) * K) {
    uint4 u[K], d[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long long q = p + static_cast<long long>(k) * lanes;
      if (q < at.p1) {
        u[k] = *(reinterpret_cast<const uint4*>(x + q * a.C) + v);
        d[k] = *(reinterpret_cast<const uint4*>(dy + q * a.C) + v);
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long long q = p + static_cast<long long>(k) * lanes;
      if (q < at.p1) {
        float f[V], h[V];
        Vec16<T>::unpack(u[k], f);
        Vec16<T>::unpack(d[k], h);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = gn_xhat(f[e], ch.mean[e], ch.rstd[e]);
          const float dz = h[e] * gn_act_grad<T>(__fmaf_rn(xh, ch.w[e], ch.b[e]), a.act, a.alpha);
          // (the product w dz rounded on its own, as in the sums: over one value it cancels
          // against its mean exactly)
          const float t = __fsub_rn(__fmul_rn(ch.w[e], dz), mz[e]);
          f[e] = ch.rstd[e] * fmaf(-xh, mx[e], t);
        }
        *(reinterpret_cast<uint4*>(dx + q * a.C) + v) = Vec16<T>::pack(f);
      }
    }
  }
}

// dbias[c] and dweight[c] from every block's row: 32 channels per block, 32 row lanes.
struct GnSumSpan {
  float* dw;  // null: not wanted
  float* db;
  int row0, rows;
};
struct GnSumArgs {
  GnSumSpan span[kGnMaxRuns];
  const float* part_c;
  int C;
};
__global__ void __launch_bounds__(1024) gn_bwd_sum_kernel(const __grid_constant__ GnSumArgs a) {
  __shared__ float s[2][32][33];
  const int blocks_c = (a.C + 31) / 32;
  const GnSumSpan sp = a.span[blockIdx.x / blocks_c];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int c = (blockIdx.x % blocks_c) * 32 + lane;
  griddep_wait();
  float z = 0.f, x = 0.f;
  if (c < a.C) {
    for (int i = row; i < sp.rows; i += 32) {
      const float* p = a.part_c + static_cast<size_t>(sp.row0 + i) * 2 * a.C;
      z += p[c];
      x += p[a.C + c];
    }
  }
  s[0][row][lane] = z;
  s[1][row][lane] = x;
  __syncthreads();
  // warp 0 adds dbias, warp 1 dweight: channel `lane`, row lanes in order
  if (row < 2 && c < a.C) {
    float t = 0.f;
    for (int i = 0; i < 32; ++i) t += s[row][i][lane];
    float* out = row == 0 ? sp.db : sp.dw;
    if (out != nullptr) out[c] = t;
  }
}

// ------------------------------------------------------------------------------ host side
// The launches of one call: runs of images whose maps together stay within `budget` bytes (one
// image at least), at most kGnMaxRuns of them per launch.
struct GnLaunch {
  std::vector<GnRun> runs;  // (x, g, y, ... filled by the caller)
  std::vector<int> level;
  int blocks = 0;
};
struct GnSchedule {
  std::vector<GnLaunch> launches;
  int rows = 0;
};

// Cuts the launch's images into chunks: about `target` blocks of equal bytes (the levels of a
// launch share them in proportion), none below 16 KB.
void gn_cut(GnLaunch& l, const std::vector<int>& images, long long pixel_bytes, int target) {
  long long total = 0;
  for (size_t i = 0; i < l.runs.size(); ++i) total += l.runs[i].pixels * pixel_bytes * images[i];
  long long per_block = std::max<long long>((total + target - 1) / target, 16384);
  for (;;) {
    long long blocks = 0;
    for (size_t i = 0; i < l.runs.size(); ++i) {
      GnRun& r = l.runs[i];
      long long per = std::max<long long>(1, per_block / pixel_bytes);
      r.chunks = static_cast<int>((r.pixels + per - 1) / per);
      r.per = (r.pixels + r.chunks - 1) / r.chunks;
      r.chunks = static_cast<int>((r.pixels + r.per - 1) / r.per);  // (none empty)
      blocks += static_cast<long long>(r.chunks) * images[i];
    }
    long long at_least = 0;
    for (int n : images) at_least += n;
    if (blocks <= std::max<long long>(target, at_least) || per_block > total) break;
    per_block += per_block / 8;  // rounding left a second, nearly empty wave
  }
}

GnSchedule gn_schedule(int levels, int N, int C, int esz, const long long* pixels, long long budget,
                       int per_sm) {
  GnSchedule s;
  const long long pixel_bytes = static_cast<long long>(C) * esz;
  const int target = sm_count() * per_sm;
  std::vector<int> images;
  long long used = 0;
  auto close = [&] {
    if (s.launches.empty() || images.empty()) return;
    GnLaunch& l = s.launches.back();
    gn_cut(l, images, pixel_bytes, target);
    for (size_t i = 0; i < l.runs.size(); ++i) {
      l.runs[i].first_block = l.blocks;
      l.runs[i].row0 = s.rows;
      l.blocks += l.runs[i].chunks * images[i];
      s.rows += l.runs[i].chunks * images[i];
    }
    images.clear();
    used = 0;
  };
  for (int lv = 0; lv < levels; ++lv) {
    const long long bytes = pixels[lv] * pixel_bytes;
    for (int n = 0; n < N;) {
      if (s.launches.empty() || images.empty()) s.launches.emplace_back();
      GnLaunch& l = s.launches.back();
      const long long room = (budget - used) / bytes;
      int take = static_cast<int>(std::min<long long>(N - n, room));
      if (take < 1 && !images.empty()) {
        close();
        continue;
      }
      take = std::max(take, 1);
      GnRun r;
      std::memset(&r, 0, sizeof(r));
      r.pixels = pixels[lv];
      r.n0 = n;
      l.runs.push_back(r);
      l.level.push_back(lv);
      images.push_back(take);
      used += bytes * take;
      n += take;
      if (static_cast<int>(l.runs.size()) == kGnMaxRuns) close();
    }
  }
  close();
  return s;
}

// Bytes of input that a run of launches keeps in L2 between its two passes.
constexpr long long kGnForwardBudget = 48LL << 20;
constexpr long long kGnBackwardBudget = 32LL << 20;  // of x; dy doubles it

GnSchedule gn_schedule_for(DType dt, int levels, int N, int C, const long long* pixels, bool backward) {
  return gn_schedule(levels, N, C, dtype_size(dt), pixels, backward ? kGnBackwardBudget : kGnForwardBudget,
                     backward ? 1 : 2);
}

size_t gn_align(size_t n) { return (n + 255) / 256 * 256; }

bool gn_sizes_ok(int levels, int N, int C, const long long* pixels, int groups) {
  if (levels < 1 || levels > kGnMaxRuns || N < 1 || C < 8 || C % 8 != 0 || C > kGnMaxChannels ||
      groups < 1 || C % groups != 0)
    return false;
  for (int l = 0; l < levels; ++l)
    if (pixels[l] < 1) return false;
  return true;
}

template <typename T>
cudaError_t gn_forward_t(const GnSchedule& sc, GnArgs& a, const GroupNormLevel* lv, cudaStream_t s) {
  LaunchOpts first, next;
  next.pdl = true;
  bool started = false;
  for (const GnLaunch& l : sc.launches) {
    a.runs = static_cast<int>(l.runs.size());
    for (int i = 0; i < a.runs; ++i) {
      GnRun r = l.runs[i];
      const GroupNormLevel& v = lv[l.level[i]];
      r.x = v.x;
      r.y = v.y;
      r.w = v.weight;
      r.b = v.bias;
      r.mean = v.mean;
      r.rstd = v.rstd;
      a.run[i] = r;
    }
    cudaError_t e = launch_ex(gn_stats_kernel<T>, dim3(l.blocks), dim3(kGnThreads), 0, s,
                              started ? next : first, 1, a);
    if (e != cudaSuccess) return e;
    started = true;
    if ((e = launch_ex(gn_apply_kernel<T>, dim3(l.blocks), dim3(kGnThreads), 0, s, next, 1, a)) !=
        cudaSuccess)
      return e;
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t gn_backward_t(const GnSchedule& sc, GnArgs& a, const GroupNormLevel* lv, int levels, int N,
                          cudaStream_t s) {
  LaunchOpts first, next;
  next.pdl = true;
  bool started = false;
  GnSumArgs sum;
  std::memset(&sum, 0, sizeof(sum));
  sum.part_c = a.part_c;
  sum.C = a.C;
  bool want_sums = false;
  for (const GnLaunch& l : sc.launches) {
    a.runs = static_cast<int>(l.runs.size());
    bool want_dx = false;
    for (int i = 0; i < a.runs; ++i) {
      GnRun r = l.runs[i];
      const GroupNormLevel& v = lv[l.level[i]];
      r.x = v.x;
      r.g = v.grad;
      r.y = v.y;
      r.w = v.weight;
      r.b = v.bias;
      r.mean = v.mean;
      r.rstd = v.rstd;
      a.run[i] = r;
      want_dx = want_dx || v.y != nullptr;
    }
    cudaError_t e = launch_ex(gn_bwd_stats_kernel<T>, dim3(l.blocks), dim3(kGnThreads), 0, s,
                              started ? next : first, 1, a);
    if (e != cudaSuccess) return e;
    started = true;
    if (want_dx && (e = launch_ex(gn_bwd_apply_kernel<T>, dim3(l.blocks), dim3(kGnThreads), 0, s, next,
                                  1, a)) != cudaSuccess)
      return e;
  }
  // Rows of a level's images follow one another over the launches, and so do the levels: a level
  // with null dweight and dbias adds its rows to the level before it.
  int spans = 0;
  int row = 0;
  for (int v = 0; v < levels; ++v) {
    int rows = 0;
    for (const GnLaunch& l : sc.launches)
      for (size_t i = 0; i < l.runs.size(); ++i)
        if (l.level[i] == v) {
          const int end = i + 1 < l.runs.size() ? l.runs[i + 1].row0 : l.runs[0].row0 + l.blocks;
          rows += end - l.runs[i].row0;
        }
    if (v == 0 || lv[v].dweight != nullptr || lv[v].dbias != nullptr) {
      GnSumSpan& sp = sum.span[spans++];
      sp.dw = lv[v].dweight;
      sp.db = lv[v].dbias;
      sp.row0 = row;
      sp.rows = 0;
      want_sums = want_sums || sp.dw != nullptr || sp.db != nullptr;
    }
    sum.span[spans - 1].rows += rows;
    row += rows;
  }
  if (!want_sums) return cudaSuccess;
  return launch_ex(gn_bwd_sum_kernel, dim3(spans * ((a.C + 31) / 32)), dim3(1024), 0, s, next, 1, sum);
}

}  // namespace

size_t group_norm_workspace_bytes(DType dt, int levels, int N, int C, const long long* pixels,
                                  int groups, bool backward) {
  if (!gn_sizes_ok(levels, N, C, pixels, groups)) return 0;
  const GnSchedule sc = gn_schedule_for(dt, levels, N, C, pixels, backward);
  const size_t rows = static_cast<size_t>(sc.rows);
  const size_t extra = backward ? rows * 2 * C : dt == DType::F32 ? rows * groups : 0;
  return gn_align(rows * groups * sizeof(float2)) + gn_align(extra * sizeof(float));
}

cudaError_t launch_group_norm(DType dt, const GroupNormLevel* lv, int levels, int N, int C,
                              const long long* pixels, int groups, float eps, int act, float alpha,
                              bool backward, void* ws, size_t ws_bytes, cudaStream_t s) {
  if (!gn_sizes_ok(levels, N, C, pixels, groups)) return cudaErrorInvalidValue;
  const GnSchedule sc = gn_schedule_for(dt, levels, N, C, pixels, backward);
  const size_t rows = static_cast<size_t>(sc.rows);
  const size_t part = gn_align(rows * groups * sizeof(float2));
  const size_t extra = backward ? rows * 2 * C : dt == DType::F32 ? rows * groups : 0;
  if (part + gn_align(extra * sizeof(float)) > ws_bytes) return cudaErrorInvalidValue;
  GnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.C = C;
  a.groups = groups;
  a.cg = C / groups;
  a.act = act;
  a.alpha = alpha;
  a.eps = eps;
  a.part = static_cast<float2*>(ws);
  (backward ? a.part_c : a.pivot) = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + part);
  switch (dt) {
    case DType::BF16:
      return backward ? gn_backward_t<__nv_bfloat16>(sc, a, lv, levels, N, s)
                      : gn_forward_t<__nv_bfloat16>(sc, a, lv, s);
    case DType::F16:
      return backward ? gn_backward_t<__half>(sc, a, lv, levels, N, s) : gn_forward_t<__half>(sc, a, lv, s);
    case DType::F32:
      return backward ? gn_backward_t<float>(sc, a, lv, levels, N, s) : gn_forward_t<float>(sc, a, lv, s);
    default:
      return cudaErrorInvalidValue;
  }
}

}  // namespace ufpn
