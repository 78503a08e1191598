// Group norm with an activation on channels-last maps, forward and backward, for one map or
// the levels of a pyramid in one call.  (Two forms of the forward: below, for maps of any size, and
// for small ones a cluster of blocks per map, further down.)
//
// Over the m = pixels * Cg values of group g of image n (Cg = C / groups adjacent channels):
//   mean = sum x / m;  var = sum (x - mean)^2 / m;  rstd = 1 / sqrt(var + eps)
//   xhat = (x - mean) * rstd;  z = xhat * weight[c] + bias[c];  y = act(z)
// and backward, with dz = dy * act'(z):
//   dbias[c] = sum dz;  dweight[c] = sum dz * xhat   (over images and pixels)
//   dx = rstd * (w dz - mean_g(w dz) - xhat * mean_g(w dz xhat))
//
// All statistics and sums are fp32.  The variance never comes from a difference of raw moments: a
// thread sums its pixels relative to the channel's median of three of them (a fixed three of the image,
// or of the block's share), so that what it subtracts is of the size of the spread, and such (count, mean,
// M2) triples merge as
//   M2_ab = M2_a + M2_b + (mean_b - mean_a)^2 n_a n_b / (n_a + n_b),
// their means taken relative to that of the group's first channel (the pivot): a mean far above the
// spread costs no digits in between, and neither does one value far from all others (relative to the
// first pixel, a value of 1e6 there left the mean 4e-5 of the spread off, and rstd 9e-6).  Every sum has a fixed order (no atomics): the same inputs
// give the same bits.
//
// The kernel moves bytes.  The batch is cut into segments whose maps stay in the 126 MB L2 cache;
// in one cooperative launch of a block per SM, eight warps of a block take the statistics of the
// segments one after the other from HBM while eight others apply the norm to the segment before,
// which they read again, from L2 as far as it still holds them (all of 70 MB, half of 250 MB): HBM reads
// and writes overlap.  A segment's blocks count themselves into a device counter when their sums are
// written; four more warps wait for the count and merge the sums for the apply warps, while these
// still work on the segment before.  Every warp keeps bulk copies in flight into a ring of its own
// in shared memory and waits for no other warp (a ring shared by eight warps cost about 800 cycles
// a 16 KB piece), and the arithmetic runs on pairs of channels (add / mul / fma on f32x2).
#include "kernels.h"
#include "ptx.cuh"
#include "vec16.cuh"

#include <algorithm>
#include <atomic>
#include <cstring>

namespace ufpn {

namespace {

constexpr int kGnWarps = 8;            // statistics warps, and as many apply warps
constexpr int kGnThreads = 32 * kGnWarps;
constexpr int kGnMergeThreads = 128;
constexpr int kGnMergeRows = 1920;     // sums of an image that a merge has in shared memory at once
constexpr int kGnMaxRuns = 8;         // runs (images of one level) per segment
constexpr int kGnMaxChannels = 2048;  // 8 per statistics thread
constexpr int kGnStage = 4096;         // one copy of a warp; backward: half of it x, half dy
constexpr int kGnK = 8;                // pixels read before their arithmetic
constexpr int kGnStatsStages = 3, kGnApplyStages = 2;  // per warp
constexpr int kDevTimeoutNorm = 0x108;

enum : int { kGnNone = 0, kGnRelu = 1, kGnLeaky = 2, kGnSwish = 3 };

// Pairs of fp32 values, one instruction for both.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // (fmaxf drops a NaN)
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Eight adjacent channels of a pixel: one 16-byte vector of a 16-bit type, two of fp32.
template <typename T>
struct Gn8 {
  static constexpr int kVecs = static_cast<int>(sizeof(T)) / 2;
  uint4 u[kVecs];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) u[i] = *(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void load_shared(uint32_t p) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(u[i].x), "=r"(u[i].y), "=r"(u[i].z), "=r"(u[i].w)
                   : "r"(p + 16 * i));
  }
  __device__ __forceinline__ void get(float2 (&f)[4]) const {  // as pairs
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      constexpr int V = Vec16<T>::V;
      float h[V];
      Vec16<T>::unpack(u[i], h);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) f[i * (V / 2) + e] = make_float2(h[2 * e], h[2 * e + 1]);
    }
  }
};
template <typename T>
__device__ __forceinline__ void gn_put(T* p, const float2 (&f)[4]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
    constexpr int V = Vec16<T>::V;
    float h[V];
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      h[2 * e] = f[i * (V / 2) + e].x;
      h[2 * e + 1] = f[i * (V / 2) + e].y;
    }
    __stcs(reinterpret_cast<uint4*>(p) + i, Vec16<T>::pack(h));  // (not read again here: x keeps the L2 cache)
  }
}

// One level: its images, each cut into `chunks` runs of `per` pixels.
struct GnRun {
  const void* x;
  const void* g;  // backward: grad_output
  void* y;        // forward: output; backward: grad_input (null: none)
  const float* w;  // [C] or null (1)
  const float* b;  // [C] or null (0)
  float* mean;     // [N][groups]: written forward (null: not wanted), read backward
  float* rstd;
  long long pixels;  // of one image
  int per, chunks;
  int first_block;  // in its segment: block of the segment's first image, chunk 0
  int row0;         // partial results of (image n, chunk c): row row0 + n * chunks + c
};
// Segments: either the images of several small levels together (one segment), or one level in
// segments of `images` images.
struct GnPhase {
  int run0, runs;
  int images, segments;
};
struct GnArgs {
  GnRun run[kGnMaxRuns];
  GnPhase phase[kGnMaxRuns];
  int phases;
  int N, C, groups, cg;
  int act;
  int apply;  // 0: only the sums (backward without dx)
  float alpha, eps;
  float2* part;   // [row][groups]: (mean - pivot, M2) forward, (sum w dz, sum w dz xhat) backward
  float* pivot;   // forward: [row of chunk 0][groups]
  float* part_c;  // backward: [row][2][C]: sum dz, sum dz xhat
  unsigned* done;  // [segments] blocks whose sums are written, zero at launch
  int* status;     // device status word
};

// 1 / (1 + exp(-z)) of a pair.  16-bit maps, whose results are rounded to 2^-9 or 2^-12, take the
// approximate 2^v and 1 / v instructions, fp32 maps the accurate exp and division.  The rounded product
// v = -z log2(e) costs |z| 2^-23.7 of exp(-z) and the instructions some 2^-22: 2^-21 of the sigmoid at |z| = 4, 2^-18.4
// at z = -40; from z = -88.7 on exp(-z) is infinite and the sigmoid 0.  The fp32 dweight and dbias take their
// terms from it too: over 2 x 100 x 152 pixels they are 1.8e-7 to 2.7e-7 off, relative to their norm, with either
// form, and the accurate one takes 236 instead of 150 us for the training pyramid (fp16, 640 x 640, four images).
__device__ __forceinline__ float gn_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float gn_inverse(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 gn_sigmoid(float2 z) {
  if constexpr (sizeof(T) == 2) {
    constexpr float kLog2E = 1.44269504088896340736f;
    const float2 v = mul2(z, both(-kLog2E));
    const float2 d = add2(make_float2(gn_exp2(v.x), gn_exp2(v.y)), both(1.f));
    return make_float2(gn_inverse(d.x), gn_inverse(d.y));
  } else {
    return make_float2(1.f / (1.f + expf(-z.x)), 1.f / (1.f + expf(-z.y)));
  }
}
template <typename T, int kAct>
__device__ __forceinline__ float2 gn_act(float2 z, float alpha) {
  if constexpr (kAct == kGnRelu) return make_float2(max_nan(z.x, 0.f), max_nan(z.y, 0.f));
  if constexpr (kAct == kGnLeaky)
    return make_float2(z.x > 0.f ? z.x : alpha * z.x, z.y > 0.f ? z.y : alpha * z.y);
  if constexpr (kAct == kGnSwish) return mul2(z, gn_sigmoid<T>(z));
  return z;
}
// dy * act'(z)
template <typename T, int kAct>
__device__ __forceinline__ float2 gn_act_grad(float2 dy, float2 z, float alpha) {
  if constexpr (kAct == kGnRelu) return make_float2(z.x > 0.f ? dy.x : 0.f, z.y > 0.f ? dy.y : 0.f);
  if constexpr (kAct == kGnLeaky)
    return make_float2(z.x > 0.f ? dy.x : alpha * dy.x, z.y > 0.f ? dy.y : alpha * dy.y);
  if constexpr (kAct == kGnSwish) {
    const float2 q = gn_sigmoid<T>(z);
    return mul2(dy, mul2(q, fma2(z, fma2(q, both(-1.f), both(1.f)), both(1.f))));
  }
  return dy;
}

struct GnSmem {
  uint8_t stats_ring[kGnWarps][kGnStatsStages * kGnStage];
  uint8_t apply_ring[kGnWarps][kGnApplyStages * kGnStage];
  // statistics: the image's medians of three pixels; a chunk's pixel lanes [lane][C] and their pixel counts
  float first[kGnMaxChannels];
  float a[kGnMaxChannels], b[kGnMaxChannels], d[kGnMaxChannels];
  float cnt[kGnThreads];  // [warp][pixel lane of the warp]
  // merge: per thread, then by group (mean, rstd; backward: the means of w dz and w dz xhat)
  float m1[kGnMergeThreads], m2[kGnMergeThreads], m3[kGnMergeThreads];
  alignas(16) float2 rows[kGnMergeRows];
  float g1[kGnMaxChannels], g2[kGnMaxChannels];
  uint64_t stats_full[kGnWarps][kGnStatsStages], apply_full[kGnWarps][kGnApplyStages];
  uint64_t ready, taken;  // g1 and g2: written; in the apply warps' registers
  int abort_flag;
  int applied;  // the apply warps have finished every segment before this one
  int go;
};

// What a warp and its threads have of a chunk.  The C / 8 vectors of a pixel are cut into `cbs`
// blocks of at most 32; warp w has block w % cbs, and of the chunk's pixels every (8 / cbs)-th batch
// of `sp`; a thread has one vector of every wl-th pixel of a batch.
struct GnLanes {
  int cbs, vb, nw, wl, sp;
  int wi;         // the warp's first batch
  int v, pl;      // vector of the pixel, pixel lane within the warp
  int v0, nv;     // the warp's vectors
  bool works, active;
  __device__ __forceinline__ GnLanes(int C, int esz, int warp, int lane, int capacity) {
    const int vc = C >> 3;
    cbs = (vc + 31) / 32;
    vb = (vc + cbs - 1) / cbs;
    nw = kGnWarps / cbs;
    wl = 32 / vb;
    sp = capacity / (vb * 8 * esz * wl) * wl;
    works = warp < cbs * nw;
    const int cb = warp % cbs;
    wi = warp / cbs;
    v0 = cb * vb;
    nv = min(vb, vc - v0);
    pl = lane / vb;
    v = v0 + lane - pl * vb;
    active = works && pl < wl && v < v0 + nv;
  }
  // this thread's pixels of a chunk of p1
  __device__ __forceinline__ int pixels(int p1) const {
    const int round = nw * sp, full = p1 / round, rest = p1 - full * round - wi * sp;
    const int part = min(max(rest, 0), sp);  // of the last round
    return full * (sp / wl) + (part > pl ? (part - pl + wl - 1) / wl : 0);
  }
  __device__ __forceinline__ int lanes() const { return nw * wl; }  // pixel lanes of a channel
  __device__ __forceinline__ int lane_index() const { return wi * wl + pl; }
  // the count of pixel lane l of channel c (as written to `cnt`)
  __device__ __forceinline__ int count_slot(int c, int l) const {
    const int i = l / wl;
    return ((c >> 3) / vb + cbs * i) * 32 + l - i * wl;
  }
};

// A chunk of the work: level, image and pixels.
struct GnPlace {
  int run, n, chunk, row;
  int p1;       // pixels of the chunk
  size_t base;  // element of the chunk's first pixel
  __device__ __forceinline__ int row_of_chunk0() const { return row - chunk; }
};
// This block's chunks in order, over all segments.
struct GnCursor {
  int phase = 0, seg = 0, block, blocks;
  int k = 0;  // segment index over all phases
  __device__ __forceinline__ explicit GnCursor(const GnArgs& a) {
    block = static_cast<int>(blockIdx.x);
    blocks = count(a);
    settle(a);
  }
  __device__ __forceinline__ bool more(const GnArgs& a) const { return phase < a.phases; }
  __device__ __forceinline__ void next(const GnArgs& a) {
    block += static_cast<int>(gridDim.x);
    settle(a);
  }
  __device__ __forceinline__ GnPlace place(const GnArgs& a) const {
    const GnPhase& ph = a.phase[phase];
    GnPlace p;
    p.run = ph.run0;
    while (p.run + 1 < ph.run0 + ph.runs && block >= a.run[p.run + 1].first_block) ++p.run;
    const GnRun& r = a.run[p.run];
    const int b = block - r.first_block;
    const int img = b / r.chunks;
    p.chunk = b - img * r.chunks;
    p.n = seg * ph.images + img;
    p.row = r.row0 + p.n * r.chunks + p.chunk;
    const long long first = static_cast<long long>(p.chunk) * r.per;
    p.base = (static_cast<size_t>(p.n) * r.pixels + first) * a.C;
    p.p1 = static_cast<int>(min(static_cast<long long>(r.per), r.pixels - first));
    return p;
  }

 private:
  __device__ __forceinline__ int count(const GnArgs& a) const {
    const GnPhase& ph = a.phase[phase];
    const GnRun& last = a.run[ph.run0 + ph.runs - 1];
    return last.first_block + min(ph.images, a.N - seg * ph.images) * last.chunks;
  }
  __device__ __forceinline__ void settle(const GnArgs& a) {  // to a segment that has this block
    while (block >= blocks) {
      block = static_cast<int>(blockIdx.x);
      ++k;
      if (++seg == a.phase[phase].segments) {
        seg = 0;
        if (++phase == a.phases) return;
      }
      blocks = count(a);
    }
  }
};

// A warp's ring of kStages copies and the batches of its chunks through it.
// kLast: the last reading of its maps, which may leave the L2 cache.  (The forward's first reading asks to
// stay, 42 against 49 us for an R50 pyramid; the backward's, of twice the bytes, does better not to: 146
// against 154 us for the training pyramid.)
template <typename T, bool kBackward, int kStages, bool kLast>
struct GnRing {
  static constexpr int kEsz = static_cast<int>(sizeof(T));
  uint8_t* buf;
  uint64_t* full;
  int stage = 0;
  uint32_t phase = 0;
  int ahead = 0;   // batches of the coming chunk already in flight
  int flying = 0;  // copies not yet waited for
  // the coming chunk: its first batch's bytes, bytes from one batch to the next, batches, pixels of the
  // last one
  const uint8_t* x;
  const uint8_t* dy;
  uint32_t stride;
  int nb, last;

  __device__ __forceinline__ void aim(const GnArgs& a, const GnPlace& at, const GnLanes& ln) {
    const int all = (at.p1 + ln.sp - 1) / ln.sp;
    nb = ln.works && all > ln.wi ? (all - ln.wi + ln.nw - 1) / ln.nw : 0;
    last = min(ln.sp, at.p1 - (ln.wi + (nb - 1) * ln.nw) * ln.sp);
    stride = static_cast<uint32_t>(ln.nw * ln.sp * a.C * kEsz);
    const GnRun& r = a.run[at.run];
    const size_t off = (at.base + static_cast<size_t>(ln.wi * ln.sp) * a.C + ln.v0 * 8) * kEsz;
    x = static_cast<const uint8_t*>(r.x) + off;
    dy = static_cast<const uint8_t*>(r.g) + off;
    ahead = 0;
  }
  __device__ __forceinline__ void load(uint8_t* dst, const uint8_t* src, uint32_t bytes, int slot) {
    bulk_load_hint(dst, src, bytes, &full[slot], kLast || kBackward ? kPolicyEvictFirst : kPolicyEvictLast);
  }
  // Starts batch i into a stage.
  __device__ __forceinline__ void issue(const GnArgs& a, const GnLanes& ln, int i, int slot) {
    const int lane = static_cast<int>(threadIdx.x) & 31;
    ++flying;
    if (ln.cbs == 1 && lane != 0) return;
    const int n = i + 1 < nb ? ln.sp : last;
    const int row = ln.nv * 8 * kEsz;
    const size_t off = static_cast<size_t>(i) * stride;
    uint8_t* const dst = buf + slot * kGnStage;
    const uint32_t bytes = static_cast<uint32_t>(n * row);
    if (lane == 0) mbar_arrive_expect_tx(&full[slot], kBackward ? 2 * bytes : bytes);
    if (ln.cbs == 1) {  // whole pixels: contiguous
      load(dst, x + off, bytes, slot);
      if constexpr (kBackward) load(dst + kGnStage / 2, dy + off, bytes, slot);
    } else {
      __syncwarp();
      for (int k = lane; k < n; k += 32) {
        const size_t o = off + static_cast<size_t>(k) * (a.C * kEsz);
        load(dst + k * row, x + o, static_cast<uint32_t>(row), slot);
        if constexpr (kBackward) load(dst + kGnStage / 2 + k * row, dy + o, static_cast<uint32_t>(row), slot);
      }
    }
  }
  // Starts the first copies of the chunk, behind those of the one before.
  __device__ __forceinline__ void prefetch(const GnArgs& a, const GnLanes& ln) {
    for (; ahead < kStages && ahead < nb; ++ahead) issue(a, ln, ahead, (stage + ahead) % kStages);
  }
  // The chunk's pixels in the ring: f(their 8 channels of x (, of dy), where they go in `out`, the thread's
  // first vector of the chunk's first pixel); K pixels are read before their arithmetic.
  template <int K, typename F>
  __device__ __forceinline__ void pixels(const GnArgs& a, const GnLanes& ln, GnSmem& s, T* out, F&& f) {
    prefetch(a, ln);
    const int row = ln.nv * 8 * kEsz, step = ln.wl * row;
    const uint32_t mine = smem_u32(buf) + static_cast<uint32_t>(ln.pl * row + (ln.v - ln.v0) * 8 * kEsz);
    const int ostep = ln.wl * a.C;
    T* o0 = out + static_cast<size_t>(ln.wi * ln.sp + ln.pl) * a.C;
    const uint32_t ostride = stride / kEsz;
    for (int i = 0; i < nb; ++i, o0 += ostride) {
      const bool ok = mbar_wait(&full[stage], phase, &s.abort_flag, a.status, kDevTimeoutNorm);
      if (!__all_sync(0xffffffffu, ok)) break;
      --flying;
      const int n = i + 1 < nb ? ln.sp : last;
      if (ln.active) {
        uint32_t p = mine + stage * kGnStage;
        T* o = o0;
        int q = ln.pl;
        for (; q + (K - 1) * ln.wl < n; q += K * ln.wl) {
          Gn8<T> v[K], d[K];
#pragma unroll
          for (int k = 0; k < K; ++k) {
            v[k].load_shared(p + k * step);
            if constexpr (kBackward) d[k].load_shared(p + k * step + kGnStage / 2);
          }
#pragma unroll
          for (int k = 0; k < K; ++k) f(v[k], d[k], o + k * ostep);
          p += K * step;
          o += K * ostep;
        }
#pragma unroll 1
        for (; q < n; q += ln.wl, p += step, o += ostep) {
          Gn8<T> v, d;
          v.load_shared(p);
          if constexpr (kBackward) d.load_shared(p + kGnStage / 2);
          f(v, d, o);
        }
      }
      __syncwarp();
      if (i + kStages < nb) issue(a, ln, i + kStages, stage);
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  }
  // (matters only after a timeout: no copy may land after the block has gone)
  __device__ __forceinline__ void drain() {
    for (; flying > 0; --flying) {
      mbar_wait_drain(&full[stage], phase);
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  }
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Barriers of the statistics threads and of the merging threads.
__device__ __forceinline__ void gn_stats_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kGnThreads) : "memory"); }
__device__ __forceinline__ void gn_merge_sync() {
  asm volatile("bar.sync 2, %0;" ::"n"(kGnMergeThreads) : "memory");
}


__device__ __forceinline__ float gn_lane_sum(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Threads per group in a block's sums over channels: a power of two up to a warp.
__device__ __forceinline__ int gn_group_width(const GnArgs& a, int threads = kGnThreads) {
  int t = 32;
  while (t > 1 && (t * a.groups > threads || t > a.cg)) t >>= 1;
  return t;
}

// A thread's 8 channels of [pixel lane][C] (two 16-byte stores).
__device__ __forceinline__ void gn_lane_store(float* dst, const float2 (&f)[4]) {
  *reinterpret_cast<float4*>(dst) = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
  *(reinterpret_cast<float4*>(dst) + 1) = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
}

// The median of three values of each channel.
template <typename T>
__device__ __forceinline__ void gn_medians(const Gn8<T>& a, const Gn8<T>& b, const Gn8<T>& c, float2 (&m)[4]) {
  float2 x[4], y[4], z[4];
  a.get(x);
  b.get(y);
  c.get(z);
  auto median = [](float u, float v, float w) { return fmaxf(fminf(u, v), fminf(fmaxf(u, v), w)); };
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = make_float2(median(x[i].x, y[i].x, z[i].x), median(x[i].y, y[i].y, z[i].y));
}

// Statistics of a chunk by group: part[row][g] = (mean - pivot, M2); the pivots are the medians of the
// group's first channel.
template <typename T, typename Ring>
__device__ __forceinline__ void gn_stats_sums(const GnArgs& a, const GnPlace& at, const GnLanes& ln,
                                              GnSmem& s, Ring& ring) {
  float2 np[4], s1[4], s2[4];  // minus the medians; sums relative to them
#pragma unroll
  for (int i = 0; i < 4; ++i) np[i] = s1[i] = s2[i] = both(0.f);
  ring.prefetch(a, ln);
  if (ln.active) {
    const GnRun& r = a.run[at.run];
    const T* image = static_cast<const T*>(r.x) + static_cast<size_t>(at.n) * r.pixels * a.C + ln.v * 8;
    Gn8<T> t[3];
    t[0].load(image);
    t[1].load(image + static_cast<size_t>(r.pixels / 2) * a.C);
    t[2].load(image + static_cast<size_t>(r.pixels - 1) * a.C);
    gn_medians(t[0], t[1], t[2], np);
    if (ln.lane_index() == 0) gn_lane_store(&s.first[ln.v * 8], np);
#pragma unroll
    for (int i = 0; i < 4; ++i) np[i] = make_float2(-np[i].x, -np[i].y);
  }
  ring.template pixels<kGnK * 2 / sizeof(T)>(
      a, ln, s, static_cast<T*>(nullptr), [&](const Gn8<T>& x, const Gn8<T>&, T*) {
        float2 f[4];
        x.get(f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 d = add2(f[i], np[i]);
          s1[i] = add2(s1[i], d);
          s2[i] = fma2(d, d, s2[i]);
        }
      });
  const int cnt = ln.pixels(at.p1);
  if (ln.active) {
    const float inv = cnt > 0 ? 1.f / static_cast<float>(cnt) : 0.f;
    float2 m[4], q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = mul2(s1[i], both(inv));
      // (rounding may leave a constant's squares below 0)
      q[i] = make_float2(max_nan(fmaf(-m[i].x, s1[i].x, s2[i].x), 0.f),
                         max_nan(fmaf(-m[i].y, s1[i].y, s2[i].y), 0.f));
      np[i] = make_float2(-np[i].x, -np[i].y);
    }
    const int o = ln.lane_index() * a.C + ln.v * 8;
    gn_lane_store(&s.d[o], np);
    gn_lane_store(&s.a[o], m);
    gn_lane_store(&s.b[o], q);
    if (ln.v == ln.v0) s.cnt[(threadIdx.x & ~31u) + ln.pl] = static_cast<float>(cnt);
  }
}
__device__ __forceinline__ void gn_stats_reduce(const GnArgs& a, const GnPlace& at, const GnLanes& ln,
                                                GnSmem& s) {
  const float px = static_cast<float>(at.p1), inv_px = 1.f / px;
  const int lanes = ln.lanes();
  // a channel's lanes: (mean - pivot, M2)
  auto channel = [&](int c, int g) {
    const float pivot = s.first[g * a.cg];
    float m = 0.f, q = 0.f;
    if (lanes == kGnWarps && ln.wl == 1) {
      float v[kGnWarps], n[kGnWarps];
#pragma unroll
      for (int l = 0; l < kGnWarps; ++l) {
        n[l] = s.cnt[l * 32];
        v[l] = (s.d[l * a.C + c] - pivot) + s.a[l * a.C + c];
        if (n[l] > 0.f) m = fmaf(n[l], v[l], m);
      }
      m *= inv_px;
#pragma unroll
      for (int l = 0; l < kGnWarps; ++l) {
        const float d = v[l] - m;
        if (n[l] > 0.f) q += fmaf(d * d, n[l], s.b[l * a.C + c]);
      }
      return make_float2(m, q);
    }
    for (int l = 0; l < lanes; ++l) {
      const float n = s.cnt[ln.count_slot(c, l)];
      if (n > 0.f) m = fmaf(n, (s.d[l * a.C + c] - pivot) + s.a[l * a.C + c], m);
    }
    m *= inv_px;
    for (int l = 0; l < lanes; ++l) {
      const float n = s.cnt[ln.count_slot(c, l)];
      const float d = ((s.d[l * a.C + c] - pivot) + s.a[l * a.C + c]) - m;
      if (n > 0.f) q += fmaf(d * d, n, s.b[l * a.C + c]);
    }
    return make_float2(m, q);
  };
  const size_t row = static_cast<size_t>(at.row) * a.groups;
  const int t = static_cast<int>(threadIdx.x);
  if (a.cg <= 32 && (a.cg & (a.cg - 1)) == 0) {
    // adjacent threads have a group's channels: merged pairwise by shuffles (equal counts)
    for (int c0 = 0; c0 < a.C; c0 += kGnThreads) {
      const int c = c0 + t, g = c / a.cg;
      float2 v = c < a.C ? channel(c, g) : both(0.f);
      float n = px;
      for (int o = 1; o < a.cg; o <<= 1, n += n) {
        const float m = __shfl_xor_sync(0xffffffffu, v.x, o), q = __shfl_xor_sync(0xffffffffu, v.y, o);
        const float d = m - v.x;
        v.x = 0.5f * (v.x + m);
        v.y = fmaf(0.5f * d * d, n, v.y + q);
      }
      if (c < a.C && c == g * a.cg) {
        a.part[row + g] = v;
        if (at.chunk == 0) a.pivot[row + g] = s.first[c];
      }
    }
    return;
  }
  for (int c = t; c < a.C; c += kGnThreads) {
    const float2 v = channel(c, c / a.cg);
    s.a[c] = v.x;  // (column c of lane 0: this thread's own)
    s.b[c] = v.y;
  }
  gn_stats_sync();
  const int width = gn_group_width(a), j = t % width;
  const float inv_cg = 1.f / static_cast<float>(a.cg);
  for (int g0 = 0; g0 < a.groups; g0 += kGnThreads / width) {
    const int g = g0 + t / width;
    const int n = g < a.groups ? a.cg : 0;
    float m = 0.f, q = 0.f;
    for (int c = j; c < n; c += width) m += s.a[g * a.cg + c];
    m = gn_lane_sum(m, width) * inv_cg;
    for (int c = j; c < n; c += width) {
      const float d = s.a[g * a.cg + c] - m;
      q += fmaf(d * d, px, s.b[g * a.cg + c]);
    }
    q = gn_lane_sum(q, width);
    if (n > 0 && j == 0) {
      a.part[row + g] = make_float2(m, q);
      if (at.chunk == 0) a.pivot[row + g] = s.first[g * a.cg];
    }
  }
}

// The merge's rows [r0, r0 + n) of groups [g0, g0 + span) into shared memory.  (One asynchronous copy after
// the other from a short loop, all in flight at once; under the streaming of the other warps a copy takes
// 2000 to 13000 cycles.)
__device__ __forceinline__ void gn_merge_fetch(const GnArgs& a, const float2* rows, int g0, int span, int r0, int n,
                                               GnSmem& s, int t) {
  const float2* src = rows + static_cast<size_t>(r0) * a.groups + g0;
  if ((a.groups & 1) == 0) {  // whole 16-byte vectors
    const uint32_t dst = smem_u32(s.rows);
    const int half = span >> 1;
    if (span == a.groups) {
#pragma unroll 1
      for (int i = t; i < n * half; i += kGnMergeThreads)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 16 * i), "l"(src + 2 * i) : "memory");
    } else {  // (spans of 128)
#pragma unroll 1
      for (int i = t; i < n * half; i += kGnMergeThreads) {
        const int r = i / (kGnMergeThreads / 2), c = 2 * (i % (kGnMergeThreads / 2));
        if (g0 + c < a.groups)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 16 * i),
                       "l"(src + static_cast<size_t>(r) * a.groups + c)
                       : "memory");
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
#pragma unroll 4
    for (int i = t; i < n * span; i += kGnMergeThreads) {
      const int r = i / span, c = i - r * span;
      if (g0 + c < a.groups) s.rows[i] = __ldcg(src + static_cast<size_t>(r) * a.groups + c);
    }
  }
  gn_merge_sync();
}
// f(row, its sums) for the rows of one thread: group g0 + lane, every per_g-th row from row j on.
template <typename F>
__device__ __forceinline__ void gn_merge_rows(const GnArgs& a, const float2* rows, int chunks, int g0, int span,
                                              int j, int lane, int per_g, GnSmem& s, int t, F&& f) {
  const int batch = kGnMergeRows / span / per_g * per_g;
  for (int r0 = 0; r0 < chunks; r0 += batch) {
    const int n = min(batch, chunks - r0);
    if (r0 > 0) gn_merge_sync();
    gn_merge_fetch(a, rows, g0, span, r0, n, s, t);
    if (j < per_g && g0 + lane < a.groups) {
#pragma unroll 2
      for (int i = j; i < n; i += per_g) f(r0 + i, s.rows[i * span + lane]);
    }
  }
}

// The image's statistics from its chunks' rows, by group: g1 = mean, g2 = rstd.  A thread sums its
// rows relative to its first one.
__device__ __forceinline__ void gn_merge_stats(const GnArgs& a, const GnPlace& at, GnSmem& s, int t) {
  const size_t row0 = static_cast<size_t>(at.row_of_chunk0()) * a.groups;
  const GnRun& r = a.run[at.run];
  const int chunks = r.chunks;
  const int span = min(a.groups, kGnMergeThreads);
  const int per_g = kGnMergeThreads / span;  // threads per group, each over every per_g-th row
  const int j = t / span, lane = t - j * span;
  const float cg = static_cast<float>(a.cg), px = static_cast<float>(r.pixels);
  const float per = static_cast<float>(r.per);
  const float tail = static_cast<float>(r.pixels - static_cast<long long>(chunks - 1) * r.per);
  for (int g0 = 0; g0 < a.groups; g0 += span) {
    const int g = g0 + lane;
    const bool in = j < per_g && g < a.groups;
    const float pivot = in && j == 0 ? __ldcg(a.pivot + row0 + g) : 0.f;
    float ref = 0.f, sd = 0.f, sq = 0.f, m2 = 0.f, cnt = 0.f;
    gn_merge_rows(a, a.part + row0, chunks, g0, span, j, lane, per_g, s, t, [&](int i, float2 v) {
      if (cnt == 0.f) ref = v.x;
      const float n = i + 1 < chunks ? per : tail;
      const float d = v.x - ref;
      sd = fmaf(n, d, sd);
      sq = fmaf(n * d, d, sq);
      m2 += v.y;
      cnt += n;
    });
    if (in) {
      const float m = cnt > 0.f ? sd / cnt : 0.f;
      s.m1[t] = ref + m;
      s.m2[t] = fmaf(cg, max_nan(fmaf(-m, sd, sq), 0.f), m2);
      s.m3[t] = cnt;
    }
    gn_merge_sync();
    if (in && j == 0) {
      float m = 0.f, q = 0.f;
#pragma unroll 4
      for (int i = 0; i < per_g; ++i)
        if (s.m3[i * span + t] > 0.f) m = fmaf(s.m3[i * span + t], s.m1[i * span + t], m);
      m /= px;
#pragma unroll 4
      for (int i = 0; i < per_g; ++i) {
        const float d = s.m1[i * span + t] - m;
        if (s.m3[i * span + t] > 0.f) q += fmaf(d * d, s.m3[i * span + t] * cg, s.m2[i * span + t]);
      }
      const float mu = m + pivot;
      const float rs = 1.f / sqrtf(q / (px * cg) + a.eps);
      s.g1[g] = mu;
      s.g2[g] = rs;
      if (at.chunk == 0 && r.mean != nullptr) {
        r.mean[static_cast<size_t>(at.n) * a.groups + g] = mu;
        r.rstd[static_cast<size_t>(at.n) * a.groups + g] = rs;
      }
    }
    gn_merge_sync();
  }
}

// A value per channel pair, of the channel's group: one for all 8 channels of a thread where groups
// are whole vectors (kWhole: Cg % 8 == 0), else one per channel.
template <bool kWhole>
struct GnByGroup {
  float2 v[kWhole ? 1 : 4];
  __device__ __forceinline__ float2 operator[](int i) const { return v[kWhole ? 0 : i]; }
  // f(group)
  template <typename F>
  __device__ __forceinline__ void set(const GnArgs& a, int vector, F&& f) {
    int g = vector * 8 / a.cg;
    if constexpr (kWhole) {
      v[0] = both(f(g));
    } else {
      int rem = vector * 8 - g * a.cg;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float t[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          t[k] = f(g);
          if (++rem == a.cg) {
            rem = 0;
            ++g;
          }
        }
        v[i] = make_float2(t[0], t[1]);
      }
    }
  }
};
// A thread's constants: z = (x - mean) * wr + b with wr = weight * rstd.  (x - mean first: no digits
// of a large mean enter the product, and a constant group gives exactly b.  The backward forms z
// with the same steps, so both take the same side of an activation's kink.)
template <bool kWhole>
struct GnChannels {
  GnByGroup<kWhole> nm;  // -mean
  float2 wr[4], b[4];
  __device__ __forceinline__ void weights(const GnRun& r, int v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wr[i] = r.w != nullptr ? make_float2(__ldg(r.w + v * 8 + 2 * i), __ldg(r.w + v * 8 + 2 * i + 1)) : both(1.f);
      b[i] = r.b != nullptr ? make_float2(__ldg(r.b + v * 8 + 2 * i), __ldg(r.b + v * 8 + 2 * i + 1)) : both(0.f);
    }
  }
  // (after weights)
  __device__ __forceinline__ void statistics(const GnArgs& a, int v, const float* mean, const float* rstd) {
    nm.set(a, v, [&](int g) { return -mean[g]; });
    GnByGroup<kWhole> rs;
    rs.set(a, v, [&](int g) { return rstd[g]; });
#pragma unroll
    for (int i = 0; i < 4; ++i) wr[i] = mul2(wr[i], rs[i]);
  }
  __device__ __forceinline__ float2 centred(float2 x, int i) const { return add2(x, nm[i]); }
  __device__ __forceinline__ float2 z(float2 d, int i) const { return fma2(d, wr[i], b[i]); }
};

template <typename T, int kAct, bool kWhole, typename Ring>
__device__ __forceinline__ void gn_apply_chunk(const GnArgs& a, const GnPlace& at, const GnLanes& ln, GnSmem& s,
                                               Ring& ring, const GnChannels<kWhole>& ch) {
  const float alpha = a.alpha;
  ring.template pixels<kGnK / sizeof(T)>(
      a, ln, s, static_cast<T*>(a.run[at.run].y) + at.base + ln.v * 8,
      [&](const Gn8<T>& x, const Gn8<T>&, T* y) {
        float2 f[4];
        x.get(f);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = gn_act<T, kAct>(ch.z(ch.centred(f[i], i), i), alpha);
        gn_put<T>(y, f);
      });
}
template <typename T, bool kWhole, typename Ring>
__device__ __forceinline__ void gn_apply(const GnArgs& a, const GnPlace& at, const GnLanes& ln, GnSmem& s,
                                         Ring& ring, const GnChannels<kWhole>& ch) {
  switch (a.act) {
    case kGnRelu: return gn_apply_chunk<T, kGnRelu>(a, at, ln, s, ring, ch);
    case kGnLeaky: return gn_apply_chunk<T, kGnLeaky>(a, at, ln, s, ring, ch);
    case kGnSwish: return gn_apply_chunk<T, kGnSwish>(a, at, ln, s, ring, ch);
    default: return gn_apply_chunk<T, kGnNone>(a, at, ln, s, ring, ch);
  }
}

// Backward sums of a chunk: by channel (part_c, for dweight / dbias) and, weighted, by group
// (part, for dx).  The pixels' sums are of dz and dz (x - mean); rstd follows at their end.
template <typename T, int kAct, bool kWhole, typename Ring>
__device__ __forceinline__ void gn_bwd_chunk_sums(const GnArgs& a, const GnPlace& at, const GnLanes& ln,
                                                  GnSmem& s, Ring& ring, const GnChannels<kWhole>& ch,
                                                  float2 (&sz)[4], float2 (&sx)[4]) {
  const float alpha = a.alpha;
  ring.template pixels<kGnK / sizeof(T)>(
      a, ln, s, static_cast<T*>(nullptr),
      [&](const Gn8<T>& x, const Gn8<T>& d, T*) {
        float2 f[4], h[4];
        x.get(f);
        d.get(h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 e = ch.centred(f[i], i);
          const float2 dz = gn_act_grad<T, kAct>(h[i], ch.z(e, i), alpha);
          sz[i] = add2(sz[i], dz);
          sx[i] = fma2(dz, e, sx[i]);
        }
      });
}
template <typename T, bool kWhole, typename Ring>
__device__ __forceinline__ void gn_bwd_sums(const GnArgs& a, const GnPlace& at, const GnLanes& ln, GnSmem& s,
                                            Ring& ring) {
  GnChannels<kWhole> ch;
  const GnRun& r = a.run[at.run];
  if (ln.active) {
    ch.weights(r, ln.v);
    ch.statistics(a, ln.v, r.mean + static_cast<size_t>(at.n) * a.groups,
                  r.rstd + static_cast<size_t>(at.n) * a.groups);
  }
  float2 sz[4], sx[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) sz[i] = sx[i] = both(0.f);
  switch (a.act) {
    case kGnRelu: gn_bwd_chunk_sums<T, kGnRelu>(a, at, ln, s, ring, ch, sz, sx); break;
    case kGnLeaky: gn_bwd_chunk_sums<T, kGnLeaky>(a, at, ln, s, ring, ch, sz, sx); break;
    case kGnSwish: gn_bwd_chunk_sums<T, kGnSwish>(a, at, ln, s, ring, ch, sz, sx); break;
    default: gn_bwd_chunk_sums<T, kGnNone>(a, at, ln, s, ring, ch, sz, sx);
  }
  if (ln.active) {
    GnByGroup<kWhole> rs;
    rs.set(a, ln.v, [&](int g) { return r.rstd[static_cast<size_t>(at.n) * a.groups + g]; });
#pragma unroll
    for (int i = 0; i < 4; ++i) sx[i] = mul2(sx[i], rs[i]);
    const int o = ln.lane_index() * a.C + ln.v * 8;
    gn_lane_store(&s.a[o], sz);
    gn_lane_store(&s.b[o], sx);
  }
}
__device__ __forceinline__ void gn_bwd_reduce(const GnArgs& a, const GnPlace& at, const GnLanes& ln, GnSmem& s) {
  float* pc = a.part_c + static_cast<size_t>(at.row) * 2 * a.C;
  const float* w = a.run[at.run].w;
  const int t = static_cast<int>(threadIdx.x), lanes = ln.lanes();
  for (int c = t; c < a.C; c += kGnThreads) {
    float z = 0.f, x = 0.f;
#pragma unroll 8
    for (int l = 0; l < lanes; ++l) {
      z += s.a[l * a.C + c];
      x += s.b[l * a.C + c];
    }
    pc[c] = z;
    pc[a.C + c] = x;
    const float wc = w != nullptr ? __ldg(w + c) : 1.f;
    s.first[c] = wc * z;
    s.d[c] = wc * x;
  }
  gn_stats_sync();
  const int width = gn_group_width(a), j = t % width;
  for (int g0 = 0; g0 < a.groups; g0 += kGnThreads / width) {
    const int g = g0 + t / width;
    const int n = g < a.groups ? a.cg : 0;
    float z = 0.f, x = 0.f;
    for (int c = j; c < n; c += width) {
      z += s.first[g * a.cg + c];
      x += s.d[g * a.cg + c];
    }
    z = gn_lane_sum(z, width);
    x = gn_lane_sum(x, width);
    if (n > 0 && j == 0) a.part[static_cast<size_t>(at.row) * a.groups + g] = make_float2(z, x);
  }
}
// The image's sums over its chunks' rows, by group: g1 = mean of w dz, g2 = mean of w dz xhat.
__device__ __forceinline__ void gn_bwd_merge(const GnArgs& a, const GnPlace& at, GnSmem& s, int t) {
  const GnRun& r = a.run[at.run];
  const float2* rows = a.part + static_cast<size_t>(at.row_of_chunk0()) * a.groups;
  const int span = min(a.groups, kGnMergeThreads);
  const int per_g = kGnMergeThreads / span;
  const int j = t / span, lane = t - j * span;
  const float inv_m = 1.f / (static_cast<float>(r.pixels) * static_cast<float>(a.cg));
  for (int g0 = 0; g0 < a.groups; g0 += span) {
    const int g = g0 + lane;
    const bool in = j < per_g && g < a.groups;
    float z = 0.f, x = 0.f;
    gn_merge_rows(a, rows, r.chunks, g0, span, j, lane, per_g, s, t, [&](int, float2 v) {
      z += v.x;
      x += v.y;
    });
    if (in) {
      s.m1[t] = z;
      s.m2[t] = x;
    }
    gn_merge_sync();
    if (in && j == 0) {
      z = x = 0.f;
      for (int i = 0; i < per_g; ++i) {
        z += s.m1[i * span + t];
        x += s.m2[i * span + t];
      }
      s.g1[g] = __fmul_rn(z, inv_m);
      s.g2[g] = __fmul_rn(x, inv_m);
    }
    gn_merge_sync();
  }
}

// A thread's constants of dx = rstd (w dz - m1 - (x - mean) rstd m2), with the group's means m1 of w
// dz and m2 of w dz xhat.  (w dz - m1 first: over one value it cancels.)
template <bool kWhole>
struct GnGradient {
  float2 w[4];
  GnByGroup<kWhole> rs, n1, n2;  // rstd, -m1, -rstd m2
  __device__ __forceinline__ void set(const GnArgs& a, const GnRun& r, int n, int v, const float* m1,
                                      const float* m2) {
    const float* rstd = r.rstd + static_cast<size_t>(n) * a.groups;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = r.w != nullptr ? make_float2(__ldg(r.w + v * 8 + 2 * i), __ldg(r.w + v * 8 + 2 * i + 1)) : both(1.f);
    rs.set(a, v, [&](int g) { return rstd[g]; });
    n1.set(a, v, [&](int g) { return -m1[g]; });
    n2.set(a, v, [&](int g) { return -rstd[g] * m2[g]; });
  }
  __device__ __forceinline__ float2 dx(float2 e, float2 dz, int i) const {
    return mul2(rs[i], fma2(e, n2[i], fma2(w[i], dz, n1[i])));
  }
};
template <typename T, int kAct, bool kWhole, typename Ring>
__device__ __forceinline__ void gn_bwd_apply_chunk(const GnArgs& a, const GnPlace& at, const GnLanes& ln,
                                                   GnSmem& s, Ring& ring, const GnChannels<kWhole>& ch,
                                                   const GnGradient<kWhole>& gr) {
  const float alpha = a.alpha;
  ring.template pixels<kGnK / 2 / sizeof(T)>(
      a, ln, s, static_cast<T*>(a.run[at.run].y) + at.base + ln.v * 8,
      [&](const Gn8<T>& x, const Gn8<T>& d, T* dx) {
        float2 f[4], h[4];
        x.get(f);
        d.get(h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 e = ch.centred(f[i], i);
          f[i] = gr.dx(e, gn_act_grad<T, kAct>(h[i], ch.z(e, i), alpha), i);
        }
        gn_put<T>(dx, f);
      });
}
template <typename T, bool kWhole, typename Ring>
__device__ __forceinline__ void gn_bwd_apply(const GnArgs& a, const GnPlace& at, const GnLanes& ln, GnSmem& s,
                                             Ring& ring, const GnChannels<kWhole>& ch,
                                             const GnGradient<kWhole>& gr) {
  switch (a.act) {
    case kGnRelu: return gn_bwd_apply_chunk<T, kGnRelu>(a, at, ln, s, ring, ch, gr);
    case kGnLeaky: return gn_bwd_apply_chunk<T, kGnLeaky>(a, at, ln, s, ring, ch, gr);
    case kGnSwish: return gn_bwd_apply_chunk<T, kGnSwish>(a, at, ln, s, ring, ch, gr);
    default: return gn_bwd_apply_chunk<T, kGnNone>(a, at, ln, s, ring, ch, gr);
  }
}

// Gives up the launch: every bounded wait of the block ends.
__device__ __forceinline__ void gn_abort(const GnArgs& a, GnSmem& s) {
  *static_cast<volatile int*>(&s.abort_flag) = 1;
  if (a.status) atomicCAS(a.status, 0, kDevTimeoutNorm);
}
__device__ __forceinline__ bool gn_aborted(GnSmem& s) { return *static_cast<volatile int*>(&s.abort_flag) != 0; }

// One thread: waits until every block's sums of segment k are written.
__device__ __forceinline__ bool gn_wait_segment(const GnArgs& a, GnSmem& s, int k, int blocks) {
  const unsigned want = static_cast<unsigned>(blocks);
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(a.done + k) : "memory");
    if (v >= want) break;
    if (gn_aborted(s)) return false;
    if (globaltimer_ns() - t0 > kWaitTimeoutNs) {
      gn_abort(a, s);
      return false;
    }
  }
  return true;
}
// Whether the statistics of segment k may be read already: at most four segments ahead of the apply
// warps, so that these find theirs in L2 (two ahead left them waiting: 129 us instead of 125 us for 8 x
// 200 x 304 x 256 bf16 with swish).
__device__ __forceinline__ bool gn_may_read(const GnArgs& a, GnSmem& s, int k) {
  return !a.apply || *static_cast<volatile int*>(&s.applied) >= k - 3;
}

// Warps 0-7: statistics; 8-15: apply; 16-19: merge.
template <typename T, bool kBackward, bool kWhole>
__global__ void __launch_bounds__(2 * kGnThreads + kGnMergeThreads, 1)
    gn_kernel(const __grid_constant__ GnArgs a) {
  extern __shared__ __align__(128) uint8_t gn_smem[];
  GnSmem& s = *reinterpret_cast<GnSmem*>(gn_smem);
  constexpr int kCapacity = kBackward ? kGnStage / 2 : kGnStage;
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kGnWarps; ++w) {
      for (int i = 0; i < kGnStatsStages; ++i) mbar_init(&s.stats_full[w][i], 1);
      for (int i = 0; i < kGnApplyStages; ++i) mbar_init(&s.apply_full[w][i], 1);
    }
    mbar_init(&s.ready, 1);
    mbar_init(&s.taken, kGnWarps);
    s.abort_flag = 0;
    s.applied = 0;
    fence_barrier_init();
  }
  __syncthreads();
  if (warp < kGnWarps) {
    const GnLanes ln(a.C, static_cast<int>(sizeof(T)), warp, lane, kCapacity);
    GnRing<T, kBackward, kGnStatsStages, false> ring;
    ring.buf = s.stats_ring[warp];
    ring.full = s.stats_full[warp];
    GnCursor cur(a);
    GnPlace at;
    if (cur.more(a)) {
      at = cur.place(a);
      ring.aim(a, at, ln);
    }
    while (cur.more(a)) {
      const uint64_t t0 = globaltimer_ns();
      while (!__all_sync(0xffffffffu, gn_may_read(a, s, cur.k) || gn_aborted(s))) {
        __nanosleep(32);
        if (globaltimer_ns() - t0 > kWaitTimeoutNs) gn_abort(a, s);
      }
      if constexpr (kBackward)
        gn_bwd_sums<T, kWhole>(a, at, ln, s, ring);
      else
        gn_stats_sums<T>(a, at, ln, s, ring);
      GnCursor nxt = cur;
      nxt.next(a);
      GnPlace then = at;
      if (nxt.more(a)) {
        then = nxt.place(a);
        ring.aim(a, then, ln);
        if (__all_sync(0xffffffffu, gn_may_read(a, s, nxt.k))) ring.prefetch(a, ln);
      }
      gn_stats_sync();
      if constexpr (kBackward)
        gn_bwd_reduce(a, at, ln, s);
      else
        gn_stats_reduce(a, at, ln, s);
      gn_stats_sync();
      if (threadIdx.x == 0)
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(a.done + cur.k) : "memory");
      cur = nxt;
      at = then;
    }
    ring.drain();
  } else if (!a.apply) {
    return;
  } else if (warp < 2 * kGnWarps) {
    const GnLanes ln(a.C, static_cast<int>(sizeof(T)), warp - kGnWarps, lane, kCapacity);
    GnRing<T, kBackward, kGnApplyStages, true> ring;
    ring.buf = s.apply_ring[warp - kGnWarps];
    ring.full = s.apply_full[warp - kGnWarps];
    uint32_t phase = 0;
    for (GnCursor cur(a); cur.more(a); cur.next(a), phase ^= 1u) {
      const GnPlace at = cur.place(a);
      const GnRun& r = a.run[at.run];
      if (warp == kGnWarps && lane == 0) *static_cast<volatile int*>(&s.applied) = cur.k;
      // (what does not depend on the other blocks, before the wait for them)
      ring.aim(a, at, ln);
      if (r.y != nullptr) ring.prefetch(a, ln);
      GnChannels<kWhole> ch;
      if (ln.active) {
        ch.weights(r, ln.v);
        if constexpr (kBackward)
          ch.statistics(a, ln.v, r.mean + static_cast<size_t>(at.n) * a.groups,
                        r.rstd + static_cast<size_t>(at.n) * a.groups);
      }
      const bool ok = mbar_wait(&s.ready, phase, &s.abort_flag, a.status, kDevTimeoutNorm);
      if (!__all_sync(0xffffffffu, ok)) break;
      GnGradient<kWhole> gr;
      if (ln.active) {
        if constexpr (kBackward)
          gr.set(a, r, at.n, ln.v, s.g1, s.g2);
        else
          ch.statistics(a, ln.v, s.g1, s.g2);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.taken);
      if constexpr (kBackward) {
        if (r.y != nullptr) gn_bwd_apply<T>(a, at, ln, s, ring, ch, gr);
      } else {
        gn_apply<T>(a, at, ln, s, ring, ch);
      }
    }
    ring.drain();
  } else {
    const int t = static_cast<int>(threadIdx.x) - 2 * kGnThreads;
    uint32_t phase = 0;
    int waited = -1;
    for (GnCursor cur(a); cur.more(a); cur.next(a), phase ^= 1u) {
      const GnPlace at = cur.place(a);
      if (t == 0) {
        bool ok = !gn_aborted(s);
        if (ok && cur.k != waited) ok = gn_wait_segment(a, s, cur.k, cur.blocks);
        // (g1 and g2 of the chunk before are in registers)
        ok = ok && mbar_wait(&s.taken, phase ^ 1u, &s.abort_flag, a.status, kDevTimeoutNorm);
        s.go = ok;
      }
      waited = cur.k;
      gn_merge_sync();
      const bool ok = *static_cast<volatile int*>(&s.go) != 0;
      if (!ok) break;
      if constexpr (kBackward)
        gn_bwd_merge(a, at, s, t);
      else
        gn_merge_stats(a, at, s, t);
      if (t == 0) mbar_arrive(&s.ready);
    }
  }
}

// ------------------------------------------------------------------ small maps
// The forward of maps that fit a cluster's shared memory: a cluster of blocks per image and level, each
// block with a share of the pixels.  The share comes in by bulk copies and stays; the block takes its
// mean and then its squares about that mean (both passes from shared memory), the blocks exchange (pivot,
// mean, M2) through distributed shared memory, and the norm is applied from there.  x is read once, and
// there are no device counters to clear and no wait across the grid.
constexpr int kGsThreads = 512;
constexpr int kGsPieces = 4;
constexpr int kGsMaxCluster = 16;
constexpr int kGsMaxLanes = 32;
constexpr int kGsMaxGroups = 128;
struct GnSmallSmem {
  float red[8 * kGsThreads];  // a pixel lane's sums [lane][C]
  float ch[kGnMaxChannels];
  // by group: the block's pivot and its mean minus that; of every block of the cluster (pivot, mean, M2)
  float pivot[kGsMaxGroups], mean[kGsMaxGroups];
  float all[3][kGsMaxCluster][kGsMaxGroups + 1];  // (+ 1: 16 blocks' sums of a group in different banks)
  float g1[kGsMaxGroups], g2[kGsMaxGroups];
  uint64_t full[kGsPieces];
  int abort_flag;
};
constexpr int kGsDataOffset = (sizeof(GnSmallSmem) + 127) / 128 * 128;
constexpr long long kGsMaxShare = 96 << 10;
static_assert(kGsDataOffset + kGsMaxShare <= 232448, "small group norm smem");

__device__ __forceinline__ void st_cluster_f32(const float* p, uint32_t rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_u32(p), rank)), "f"(v) : "memory");
}

// The pixels q = pl, pl + lanes, .. below cnt: f(its 8 channels, pixel).
template <typename T, typename F>
__device__ __forceinline__ void gn_small_pixels(uint32_t mine, int row, int pl, int lanes, int begin, int end, F&& f) {
#pragma unroll 4
  for (int q = begin + pl; q < end; q += lanes) {
    Gn8<T> t;
    t.load_shared(mine + static_cast<uint32_t>(q) * row);
    f(t, q);
  }
}
template <typename T, int kAct, bool kWhole>
__device__ __forceinline__ void gn_small_apply(uint32_t mine, int row, int pl, int lanes, int cnt, T* y, int C,
                                               float alpha, const GnChannels<kWhole>& ch) {
  gn_small_pixels<T>(mine, row, pl, lanes, 0, cnt, [&](const Gn8<T>& x, int q) {
    float2 f[4];
    x.get(f);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = gn_act<T, kAct>(ch.z(ch.centred(f[i], i), i), alpha);
    gn_put<T>(y + static_cast<size_t>(q) * C, f);
  });
}

template <typename T, bool kWhole>
__global__ void __launch_bounds__(kGsThreads, 1) gn_small_kernel(const __grid_constant__ GnArgs a, const int log_blocks) {
  extern __shared__ __align__(128) uint8_t gs_smem[];
  GnSmallSmem& s = *reinterpret_cast<GnSmallSmem*>(gs_smem);
  const uint32_t data = smem_u32(gs_smem) + kGsDataOffset;
  const T* const first_pixel = reinterpret_cast<const T*>(gs_smem + kGsDataOffset);
  const int t = static_cast<int>(threadIdx.x);
  const int blocks = 1 << log_blocks;
  const int rank = static_cast<int>(blockIdx.x) & (blocks - 1), item = static_cast<int>(blockIdx.x) >> log_blocks;
  const GnRun& r = a.run[item / a.N];
  const int n = item % a.N;
  const int row = a.C * static_cast<int>(sizeof(T));
  const int pixels = static_cast<int>(r.pixels);
  const int first = rank * r.per, cnt = max(min(r.per, pixels - first), 0);
  const size_t base = (static_cast<size_t>(n) * pixels + first) * a.C;
  const int piece = (cnt + kGsPieces - 1) / kGsPieces;  // pixels of a copy
  if (t == 0) {
    for (int i = 0; i < kGsPieces; ++i) mbar_init(&s.full[i], 1);
    s.abort_flag = 0;
    fence_barrier_init();
    for (int i = 0; i * piece < cnt; ++i) {
      const uint32_t bytes = static_cast<uint32_t>(min(piece, cnt - i * piece) * row);
      mbar_arrive_expect_tx(&s.full[i], bytes);
      bulk_load(gs_smem + kGsDataOffset + i * piece * row,
                static_cast<const uint8_t*>(r.x) + (base * sizeof(T) + static_cast<size_t>(i) * piece * row), bytes,
                &s.full[i]);
    }
  }
  const int vc = a.C >> 3;
  const int lanes = min(kGsThreads / vc, kGsMaxLanes);
  const int pl = t / vc, v = t - pl * vc;
  const bool active = pl < lanes;
  const uint32_t mine = data + static_cast<uint32_t>(v * 8 * sizeof(T));
  GnChannels<kWhole> ch;
  if (active) ch.weights(r, v);
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (this block has started)

  // The block's mean by group, relative to the medians of three pixels of its first piece (that of the group's
  // first channel: the pivot).
  const int mid = max(piece - 1, 0) / 2, last = max(min(piece, cnt) - 1, 0);
  bool ok = true;
  float2 acc[4], p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = p[i] = both(0.f);
  for (int i = 0; i * piece < cnt; ++i) {
    ok = mbar_wait(&s.full[i], 0, &s.abort_flag, a.status, kDevTimeoutNorm) && ok;
    if (i == 0) {
      Gn8<T> f[3];
      f[0].load_shared(mine);
      f[1].load_shared(mine + static_cast<uint32_t>(mid) * row);
      f[2].load_shared(mine + static_cast<uint32_t>(last) * row);
      gn_medians(f[0], f[1], f[2], p);
    }
    if (active)
      gn_small_pixels<T>(mine, row, pl, lanes, i * piece, min(cnt, (i + 1) * piece), [&](const Gn8<T>& x, int) {
        float2 f[4];
        x.get(f);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = add2(acc[k], make_float2(f[k].x - p[k].x, f[k].y - p[k].y));
      });
  }
  // (a timeout has set the status word; the block goes on to the cluster's barriers, with no copy in flight)
  if (!ok && t == 0)
    for (int i = 0; i * piece < cnt; ++i) mbar_wait_drain(&s.full[i], 0);
  // The threads' sums over the pixel lanes, then store(group, f(channel, that) summed over its channels).
  const bool pow2 = a.cg <= 32 && (a.cg & (a.cg - 1)) == 0;
  const int width = min(gn_group_width(a, kGsThreads), 32), j = t % width;
  auto sums = [&](auto&& f, auto&& store) {
    if (active) gn_lane_store(&s.red[pl * a.C + v * 8], acc);
    __syncthreads();
    for (int c0 = 0; c0 < a.C; c0 += kGsThreads) {
      const int c = c0 + t;
      float z = 0.f;
      if (c < a.C) {
#pragma unroll 8
        for (int l = 0; l < lanes; ++l) z += s.red[l * a.C + c];
        z = f(c, z);
      }
      if (pow2) {  // adjacent threads have a group's channels
        z = gn_lane_sum(z, a.cg);
        if (c < a.C && (c & (a.cg - 1)) == 0) store(c / a.cg, z);
      } else if (c < a.C) {
        s.ch[c] = z;
      }
    }
    __syncthreads();
    if (pow2) return;
    for (int g0 = 0; g0 < a.groups; g0 += kGsThreads / width) {
      const int g = g0 + t / width, m = g < a.groups ? a.cg : 0;
      float z = 0.f;
      for (int c = j; c < m; c += width) z += s.ch[g * a.cg + c];
      z = gn_lane_sum(z, width);
      if (m > 0 && j == 0) store(g, z);
    }
    __syncthreads();
  };
  auto median = [&](int c) {
    const float u = to_float(first_pixel[c]), v = to_float(first_pixel[mid * a.C + c]),
                w = to_float(first_pixel[last * a.C + c]);
    return fmaxf(fminf(u, v), fminf(fmaxf(u, v), w));
  };
  const float inv_cnt = cnt > 0 ? 1.f / static_cast<float>(cnt) : 0.f;
  const float inv_cg = 1.f / static_cast<float>(a.cg);
  sums(
      [&](int c, float z) {
        if (cnt == 0) return 0.f;
        const int c0 = pow2 ? c & ~(a.cg - 1) : c - c % a.cg;
        return (median(c) - median(c0)) + z * inv_cnt;
      },
      [&](int g, float z) {
        s.pivot[g] = cnt > 0 ? median(g * a.cg) : 0.f;
        s.mean[g] = z * inv_cg;
      });
  // Its squares about that mean.
  {
    GnByGroup<kWhole> np, nm;
    if (active) {
      np.set(a, v, [&](int g) { return -s.pivot[g]; });
      nm.set(a, v, [&](int g) { return -s.mean[g]; });
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = both(0.f);
    if (active)
      gn_small_pixels<T>(mine, row, pl, lanes, 0, cnt, [&](const Gn8<T>& x, int) {
        float2 f[4];
        x.get(f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 d = add2(add2(f[k], np[k]), nm[k]);
          acc[k] = fma2(d, d, acc[k]);
        }
      });
  }
  sums([](int, float z) { return z; }, [&](int g, float z) { s.all[2][rank][g] = z; });
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // (every block has started)
  for (int i = t; i < blocks << 7; i += kGsThreads) {  // its sums to every block
    const int to = i / kGsMaxGroups, g = i % kGsMaxGroups;
    if (g < a.groups) {
      st_cluster_f32(&s.all[0][rank][g], to, s.pivot[g]);
      st_cluster_f32(&s.all[1][rank][g], to, s.mean[g]);
      if (to != rank) st_cluster_f32(&s.all[2][rank][g], to, s.all[2][rank][g]);
    }
  }
  __syncwarp();
  cluster_sync_all();

  // The image's statistics: a group's 16 threads have a block each.
  for (int i = t; i < (a.groups + 1) / 2 * (2 * kGsMaxCluster); i += kGsThreads) {
    const int g = min(i / kGsMaxCluster, a.groups - 1), b = i % kGsMaxCluster;
    const float share = b < blocks ? static_cast<float>(max(min(r.per, pixels - b * r.per), 0)) : 0.f;
    const float px = static_cast<float>(pixels), cg = static_cast<float>(a.cg);
    const float pivot = s.all[0][0][g];
    const float m = share > 0.f ? (s.all[0][b][g] - pivot) + s.all[1][b][g] : 0.f;
    const float mean = gn_lane_sum(share * m, kGsMaxCluster) / px;
    const float d = m - mean;
    const float m2 = gn_lane_sum(share > 0.f ? fmaf(d * d, share * cg, s.all[2][b][g]) : 0.f, kGsMaxCluster);
    if (b == 0) {
      const float mu = mean + pivot;
      const float rs = 1.f / sqrtf(m2 / (px * cg) + a.eps);
      s.g1[g] = mu;
      s.g2[g] = rs;
      if (rank == 0 && r.mean != nullptr) {
        r.mean[static_cast<size_t>(n) * a.groups + g] = mu;
        r.rstd[static_cast<size_t>(n) * a.groups + g] = rs;
      }
    }
  }
  __syncthreads();
  if (active) {
    ch.statistics(a, v, s.g1, s.g2);
    T* y = static_cast<T*>(r.y) + base + v * 8;
    switch (a.act) {
      case kGnRelu: gn_small_apply<T, kGnRelu>(mine, row, pl, lanes, cnt, y, a.C, a.alpha, ch); break;
      case kGnLeaky: gn_small_apply<T, kGnLeaky>(mine, row, pl, lanes, cnt, y, a.C, a.alpha, ch); break;
      case kGnSwish: gn_small_apply<T, kGnSwish>(mine, row, pl, lanes, cnt, y, a.C, a.alpha, ch); break;
      default: gn_small_apply<T, kGnNone>(mine, row, pl, lanes, cnt, y, a.C, a.alpha, ch);
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
#pragma unroll 4
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
struct GnSchedule {
  GnRun run[kGnMaxRuns];  // sizes only
  GnPhase phase[kGnMaxRuns];
  int phases = 0, segments = 0, blocks = 0;  // blocks: of the largest segment
  long long rows = 0;
};

// Cuts the images of a segment into chunks: about `target` blocks of equal bytes (the levels share
// them in proportion), none below 8 KB.
void gn_cut(GnRun* run, int runs, int images, long long pixel_bytes, int target) {
  long long total = 0;
  for (int i = 0; i < runs; ++i) total += run[i].pixels * pixel_bytes * images;
  long long per_block = std::max<long long>((total + target - 1) / target, 8192);
  for (;;) {
    long long blocks = 0;
    for (int i = 0; i < runs; ++i) {
      GnRun& r = run[i];
      const long long per = std::min<long long>(std::max<long long>(1, per_block / pixel_bytes), 1 << 30);
      long long chunks = (r.pixels + per - 1) / per;
      r.per = static_cast<int>((r.pixels + chunks - 1) / chunks);
      r.chunks = static_cast<int>((r.pixels + r.per - 1) / r.per);  // (none empty)
      r.first_block = static_cast<int>(blocks);
      blocks += static_cast<long long>(r.chunks) * images;
    }
    if (blocks <= std::max<long long>(target, static_cast<long long>(images) * runs) || per_block > total) break;
    per_block += per_block / 16 + 1;  // rounding left a few chunks for a second round
  }
}

GnSchedule gn_schedule(DType dt, int levels, int N, int C, const long long* pixels, long long budget) {
  GnSchedule s;
  std::memset(s.run, 0, sizeof(s.run));
  const long long pixel_bytes = static_cast<long long>(C) * dtype_size(dt);
  const int target = sm_count();
  for (int lv = 0; lv < levels;) {
    GnPhase& p = s.phase[s.phases++];
    p.run0 = lv;
    long long used = 0;
    int end = lv;
    while (end < levels && used + pixels[end] * pixel_bytes * N <= budget) used += pixels[end++] * pixel_bytes * N;
    if (end > lv) {  // whole levels together
      p.runs = end - lv;
      p.images = N;
    } else {
      p.runs = 1;
      p.images = static_cast<int>(std::max<long long>(1, budget / (pixels[lv] * pixel_bytes)));
      // (segments of equal size)
      const int count = (N + p.images - 1) / p.images;
      p.images = (N + count - 1) / count;
    }
    p.segments = (N + p.images - 1) / p.images;
    for (int i = 0; i < p.runs; ++i) s.run[lv + i].pixels = pixels[lv + i];
    gn_cut(s.run + lv, p.runs, p.images, pixel_bytes, target);
    for (int i = 0; i < p.runs; ++i) {
      s.run[lv + i].row0 = static_cast<int>(s.rows);
      s.rows += static_cast<long long>(s.run[lv + i].chunks) * N;
    }
    const GnRun& last = s.run[lv + p.runs - 1];
    s.blocks = std::max(s.blocks, last.first_block + p.images * last.chunks);
    s.segments += p.segments;
    lv += p.runs;
  }
  return s;
}

// Segment size: bytes of x (the backward's come with dy).  A segment is read again from L2 while the
// next ones stream in, so a few of them ought to fit its 126 MB; half the size reads less from HBM, but
// waits more often (the training pyramid 148 -> 152 us, the others within 1 %), twice the size costs 7 %.
constexpr long long kGnForwardBudget = 64LL << 20;
constexpr long long kGnBackwardBudget = 32LL << 20;

GnSchedule gn_schedule_for(DType dt, int levels, int N, int C, const long long* pixels, bool backward) {
  return gn_schedule(dt, levels, N, C, pixels, backward ? kGnBackwardBudget : kGnForwardBudget);
}

size_t gn_align(size_t n) { return (n + 255) / 256 * 256; }

bool gn_sizes_ok(int levels, int N, int C, const long long* pixels, int groups) {
  if (levels < 1 || levels > kGnMaxRuns || N < 1 || C < 8 || C % 8 != 0 || C > kGnMaxChannels ||
      groups < 1 || C % groups != 0)
    return false;
  // (no map beyond 2^39 values: every product of the schedule stays inside its type)
  for (int l = 0; l < levels; ++l)
    if (pixels[l] < 1 || pixels[l] > (1LL << 39) / N / C) return false;
  return true;
}

// Workspace: counters, rows by group, then pivots (forward) or rows by channel (backward).
struct GnWorkspace {
  size_t part, extra, total;
};
GnWorkspace gn_workspace(const GnSchedule& sc, int C, int groups, bool backward) {
  const size_t rows = static_cast<size_t>(sc.rows);
  GnWorkspace w;
  w.part = gn_align(sc.segments * sizeof(unsigned));
  w.extra = w.part + gn_align(rows * groups * sizeof(float2));
  w.total = w.extra + gn_align(rows * (backward ? 2 * C : groups) * sizeof(float));
  return w;
}

template <typename T, bool kBackward, bool kWhole>
cudaError_t gn_launch(const GnSchedule& sc, const GnArgs& a, cudaStream_t s) {
  const auto kernel = gn_kernel<T, kBackward, kWhole>;
  constexpr int kSmem = static_cast<int>(sizeof(GnSmem));
  static_assert(kSmem <= 232448, "group norm smem");
  static std::atomic<bool> configured[64];
  cudaError_t e = once_per_device(configured, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (e != cudaSuccess) return e;
  if ((e = cudaMemsetAsync(a.done, 0, sc.segments * sizeof(unsigned), s)) != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min(sc.blocks, sm_count())));
  cfg.blockDim = dim3(2 * kGnThreads + kGnMergeThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;  // blocks wait for one another: all resident or none
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// dweight and dbias from the rows: a level's rows follow one another, and so do the levels; one
// with null dweight and dbias adds its rows to the level before it.
cudaError_t gn_sum_rows(const GnSchedule& sc, const GnArgs& a, const GroupNormLevel* lv, int levels,
                        cudaStream_t s) {
  GnSumArgs sum;
  std::memset(&sum, 0, sizeof(sum));
  sum.part_c = a.part_c;
  sum.C = a.C;
  bool wanted = false;
  int spans = 0;
  for (int v = 0; v < levels; ++v) {
    if (v == 0 || lv[v].dweight != nullptr || lv[v].dbias != nullptr) {
      GnSumSpan& sp = sum.span[spans++];
      sp.dw = lv[v].dweight;
      sp.db = lv[v].dbias;
      sp.row0 = sc.run[v].row0;
      wanted = wanted || sp.dw != nullptr || sp.db != nullptr;
    }
    sum.span[spans - 1].rows += sc.run[v].chunks * a.N;
  }
  if (!wanted) return cudaSuccess;
  return launch_ex(gn_bwd_sum_kernel, dim3(spans * ((a.C + 31) / 32)), dim3(1024), 0, s, LaunchOpts(), 1,
                   sum);
}

template <typename T>
cudaError_t gn_run(const GnSchedule& sc, const GnArgs& a, const GroupNormLevel* lv, int levels,
                   bool backward, cudaStream_t s) {
  const bool whole = a.cg % 8 == 0;
  if (!backward) return whole ? gn_launch<T, false, true>(sc, a, s) : gn_launch<T, false, false>(sc, a, s);
  const cudaError_t e = whole ? gn_launch<T, true, true>(sc, a, s) : gn_launch<T, true, false>(sc, a, s);
  return e == cudaSuccess ? gn_sum_rows(sc, a, lv, levels, s) : e;
}

template <typename K>
cudaError_t gn_small_attributes(K kernel) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kGsDataOffset + static_cast<int>(kGsMaxShare));
  return e != cudaSuccess ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}
// Whether the current device can hold a cluster of 2^log_blocks of the small kernel's blocks with the largest
// share (a part of a GPU may have no 16 SMs in one cluster's reach).  One answer for all its types: every
// block takes an SM.  Without an answer: yes, and the launch tells.
bool gn_small_fits(int log_blocks) {
  static std::atomic<int> known[64][5];  // 0: not asked yet, 1: no, 2: yes
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return true;
  }
  int answer = known[dev][log_blocks].load(std::memory_order_relaxed);
  if (answer == 0) {
    const auto kernel = gn_small_kernel<__nv_bfloat16, true>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << log_blocks);
    cfg.blockDim = dim3(kGsThreads);
    cfg.dynamicSmemBytes = kGsDataOffset + static_cast<size_t>(kGsMaxShare);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << log_blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (gn_small_attributes(kernel) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return true;
    }
    answer = clusters > 0 ? 2 : 1;
    known[dev][log_blocks].store(answer, std::memory_order_relaxed);
  }
  return answer == 2;
}

// The small kernel's cluster size for these maps, 0 where it does not apply: shares of about 16 KB (8 and
// 32 KB measure the same), in one wave of clusters.  (A cluster's SMs lie in one GPC, so that not all 148
// can be used: 16 clusters of 8 took two waves, 18.5 us against 10.4 us for 8 of them.)  Against the
// cooperative kernel, bf16, C = 256, 32 groups: one pixel 6.3 / 10.4 us, 7 x 7 8.3 / 10.5, one to eight of
// 25 x 38 10.4 / 12.4, four of 50 x 50 (80 KB a block) 12.4 / 14.1; two of 50 x 76 at 122 KB a block would
// take 14.4 / 12.5.
int gn_small_blocks(DType dt, int levels, int N, int C, const long long* pixels, int groups) {
  if (groups > kGsMaxGroups || static_cast<long long>(N) * levels > 128) return 0;
  const long long row = static_cast<long long>(C) * dtype_size(dt);
  const int items = N * levels;
  long long most = 0;
  for (int l = 0; l < levels; ++l) most = std::max(most, pixels[l]);
  if (most > kGsMaxCluster * kGsMaxShare / row) return 0;
  int blocks = 1;
  while (blocks < kGsMaxCluster && (most + blocks - 1) / blocks * row > (16 << 10)) blocks *= 2;
  while (blocks > 1 && items * blocks > (blocks >= 8 ? 64 : 128)) blocks /= 2;
  int log_blocks = 0;
  while ((1 << log_blocks) < blocks) ++log_blocks;
  while (log_blocks > 0 && !gn_small_fits(log_blocks)) blocks = 1 << --log_blocks;
  return (most + blocks - 1) / blocks * row <= kGsMaxShare ? blocks : 0;
}
template <typename T, bool kWhole>
cudaError_t gn_small_launch(GnArgs& a, int levels, int blocks, cudaStream_t s) {
  const auto kernel = gn_small_kernel<T, kWhole>;
  static std::atomic<bool> configured[64];
  const cudaError_t e = once_per_device(configured, [&] { return gn_small_attributes(kernel); });
  if (e != cudaSuccess) return e;
  int share = 0, log_blocks = 0;
  while ((1 << log_blocks) < blocks) ++log_blocks;
  for (int l = 0; l < levels; ++l) {
    a.run[l].per = static_cast<int>((a.run[l].pixels + blocks - 1) / blocks);
    share = std::max(share, a.run[l].per);
  }
  return launch_ex(kernel, dim3(static_cast<unsigned>(levels * a.N * blocks)), dim3(kGsThreads),
                   kGsDataOffset + static_cast<size_t>(share) * a.C * sizeof(T), s, LaunchOpts(), blocks, a, log_blocks);
}
template <typename T>
cudaError_t gn_small_run(GnArgs& a, int levels, int blocks, cudaStream_t s) {
  return a.cg % 8 == 0 ? gn_small_launch<T, true>(a, levels, blocks, s) : gn_small_launch<T, false>(a, levels, blocks, s);
}

}  // namespace

size_t group_norm_workspace_bytes(DType dt, int levels, int N, int C, const long long* pixels,
                                  int groups, bool backward) {
  if (!gn_sizes_ok(levels, N, C, pixels, groups)) return kGroupNormNoSizes;
  if (!backward && gn_small_blocks(dt, levels, N, C, pixels, groups) > 0) return 0;
  const GnSchedule sc = gn_schedule_for(dt, levels, N, C, pixels, backward);
  return sc.rows < (1LL << 31) ? gn_workspace(sc, C, groups, backward).total : kGroupNormNoSizes;
}

cudaError_t launch_group_norm(DType dt, const GroupNormLevel* lv, int levels, int N, int C,
                              const long long* pixels, int groups, float eps, int act, float alpha,
                              bool backward, void* ws, size_t ws_bytes, int* status,
                              cudaStream_t s) {
  if (!gn_sizes_ok(levels, N, C, pixels, groups)) return cudaErrorInvalidValue;
  GnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.N = N;
  a.C = C;
  a.groups = groups;
  a.cg = C / groups;
  a.act = act;
  a.alpha = alpha;
  a.eps = eps;
  a.status = status;
  auto maps = [&] {
    for (int l = 0; l < levels; ++l) {
      a.run[l].x = lv[l].x;
      a.run[l].g = lv[l].grad;
      a.run[l].y = lv[l].y;
      a.run[l].w = lv[l].weight;
      a.run[l].b = lv[l].bias;
      a.run[l].mean = lv[l].mean;
      a.run[l].rstd = lv[l].rstd;
      a.run[l].pixels = pixels[l];
      a.apply |= lv[l].y != nullptr;
    }
  };
  const int small = backward ? 0 : gn_small_blocks(dt, levels, N, C, pixels, groups);
  if (small > 0) {
    maps();
    switch (dt) {
      case DType::BF16:
        return gn_small_run<__nv_bfloat16>(a, levels, small, s);
      case DType::F16:
        return gn_small_run<__half>(a, levels, small, s);
      case DType::F32:
        return gn_small_run<float>(a, levels, small, s);
      default:
        return cudaErrorInvalidValue;
    }
  }
  const GnSchedule sc = gn_schedule_for(dt, levels, N, C, pixels, backward);
  if (sc.rows >= (1LL << 31)) return cudaErrorInvalidValue;
  const GnWorkspace w = gn_workspace(sc, C, groups, backward);
  if (w.total > ws_bytes) return cudaErrorInvalidValue;
  std::memcpy(a.run, sc.run, sizeof(a.run));
  maps();
  std::memcpy(a.phase, sc.phase, sizeof(a.phase));
  a.phases = sc.phases;
  uint8_t* base = static_cast<uint8_t*>(ws);
  a.done = reinterpret_cast<unsigned*>(base);
  a.part = reinterpret_cast<float2*>(base + w.part);
  (backward ? a.part_c : a.pivot) = reinterpret_cast<float*>(base + w.extra);
  switch (dt) {
    case DType::BF16:
      return gn_run<__nv_bfloat16>(sc, a, lv, levels, backward, s);
    case DType::F16:
      return gn_run<__half>(sc, a, lv, levels, backward, s);
    case DType::F32:
      return gn_run<float>(sc, a, lv, levels, backward, s);
    default:
      return cudaErrorInvalidValue;
  }
}

}  // namespace ufpn
