// Lateral 1x1 convs with a low-rank adapter per image, forward and backward.
//
// Image n of the batch carries adapter a = index[n] (outside 0 .. L-1: none) of rank R, a pair
// down[a] [R][K], up[a] [256][R] and a scale s:
//   h = s x down[a]^T                                   [pixels][R]
//   out = x W^T + b + h up[a]^T (+ bilinear(coarse))    [pixels][256]
// and backward, with dy the gradient of out:
//   dh = s dy up[a];  dx = dy W + dh down[a]
//   ddown[a] = sum over the images of a of dh^T x;  dup[a] = sum of dy^T h
//
// fpn_adapter_kernel computes out (and, with the transposed operands, dx) in one pass over x: the
// k-loop of the shared projection feeds every x tile to two tcgen05.mma, N = 256 columns of W and
// N = R columns of down[a]; h leaves TMEM through the epilogue warps, which scale it and put it
// back into shared memory as the A operand of a last MMA against up[a], on the accumulator that
// already holds x W^T.  So an adapter costs R / 256 more tensor work and no further pass.
//
// h is kept in 16-bit parts, hi = round(h), the next = round(h - hi) and so on: three of bf16 carry 22
// bits and more, two of fp16 as many down to |h| = 2^-3 and whatever lies above 2^-25 below that (there
// the second part is subnormal).  For out and dx that is enough: fp16 results have steps of 2^-24
// themselves.  The weight gradients are fp32, and dh is as small as up and dy make it, so their GEMM, which
// can weigh each part's columns when it adds them, takes other parts of fp16: dh / 2, then
// what is left times 2^10 and times 2^22 (all bits down to 2^-47), and for h the bits that the second part
// lost times 2^11 (down to 2^-36) as a third part.  (With two plain parts ddown was 1e-3 off at dy and up
// of 1e-3, 0.37 at 3e-5 and 1e-4.)
// One rounding to bf16 would be the largest error of the fp32 weight gradients, and of an adapter's share
// of out; the further parts cost one k-step of the last MMA each, and columns of the gradients'
// GEMM.  The tensor cores' fp32 accumulation rounds every step
// downwards, an error that grows with the number of steps: the products behind h are split over up to
// four accumulators (32 steps each at K = 2048: dup 3.1e-6 -> 0.8e-6 off at fp16).
#include "kernels.h"
#include "tc_gemm.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

namespace ufpn {

namespace {

constexpr int kAdMaxRank = 64;
// TMA warp, MMA warp, 16 epilogue warps: what the epilogue does for a tile is one long chain of
// instructions, so that twice the warps halve its time (8 warps: about 6000 cycles a tile).  On P2 of eight
// images, 144 us, a tile takes 10000 cycles: h and its parts 2000, the last MMA and the accumulators' reading
// 1500, stores 4700, the next top-down weights 1200.  Four more warps that make h and those weights while
// the others store took 154 us (118 instead of 122 without a top-down add): the k-loop then waits for
// loads, x from HBM and the 128 KB of weights that every tile reads again from L2.  (These times and the others
// of P2 in this file are of the same maps pass after pass, of which L2 keeps a part: a call whose maps are
// new takes 156 to 167 us, and choices that lie a few percent apart were not compared there.)
constexpr int kAdEpiWarps = 16;
constexpr int kAdThreads = 64 + 32 * kAdEpiWarps;
constexpr int kAdWarpCols = kTcBlockN / (kAdEpiWarps / 4);  // output channels of a warp
constexpr int kDevTimeoutAdapter = 0x107;

template <typename T>
constexpr int kAdParts = TcElem<T>::kFmt == 1 ? 3 : 2;  // of h in the last MMA: bf16, fp16
constexpr int kAdStored = 3;                            // of h and dh as stored for the gradients, at most

// K-major operand rows of RB = 32, 64 or 128 bytes under the swizzle of that width (16-byte chunk c of
// row r at c ^ (r * RB / 128 % (RB / 16))), 8-row atoms of 8 RB bytes.
template <int RB>
__device__ __forceinline__ uint64_t sdesc_kmajor_rows(uint32_t saddr) {
  constexpr uint64_t layout = RB == 128 ? 2 : RB == 64 ? 4 : 6;
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1) << 16;
  d |= static_cast<uint64_t>(8 * RB >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= layout << 61;
  return d;
}
template <int RB>
__device__ __forceinline__ uint32_t row_chunk(int row, int chunk) {
  return static_cast<uint32_t>(row * RB + ((chunk ^ ((row * RB / 128) & (RB / 16 - 1))) << 4));
}

// Shared memory of fpn_adapter_kernel for ranks up to RP.  (Keeping 256 x 256 weights resident instead
// of streaming them with every tile changed nothing: 148 against 146 us on P2 of eight images, the same
// maps pass after pass.)
template <int RP, int kParts, bool kTaps>
struct AdCfg {
  static constexpr int kRow = RP * 2;   // bytes of a row of h or up
  static constexpr int kU = RP * 128;   // one k-block of down[a]
  static constexpr int kOffU = kTcAStage + kTcBStage;
  static constexpr int kStage = kOffU + kU;
  static constexpr int kStages = RP <= 32 ? 3 : 2;  // (three of 56 KB would not fit)
  static constexpr int kPart = kTcBlockM * kRow;
  // h's parts; before them, in the same place, the top-down weights in up to two parts (their MMA is over when
  // h is)
  static constexpr int kT = kTaps || kParts * kPart > 2 * kTcAStage ? kParts * kPart : 2 * kTcAStage;
  static constexpr int kStaging = 1024;  // per epilogue warp: 8 pixels x 64 channels
  static constexpr int kOffV = kStages * kStage;  // up[a]: 256 rows
  static constexpr int kOffT = kOffV + kTcBlockN * kRow;
  static constexpr int kOffStaging = kOffT + kT;
  static constexpr int kOffBias = kOffStaging + kAdEpiWarps * kStaging;
  static constexpr int kOffBars = kOffBias + kTcBlockN * 4;
  static constexpr int kSmemBytes = kOffBars + 256 + 1024 /*alignment slack*/;
  static_assert(kU % 1024 == 0 && kPart % 1024 == 0 && kT % 1024 == 0 && kSmemBytes <= 232448, "adapter smem");
};

struct AdArgs {
  const int* index;     // [N]
  const float* scales;  // [L] or null (1)
  float scale;
  int adapters, rank;
  // element (a, output channel c, r) of the last MMA's B operand: v + a * va + c * vc + r * vr
  const void* v;
  long long va, vc, vr;
  int v_rows;    // output channels
  int v_vec;     // vr == 1 and every row is whole 16-byte vectors
  void* hidden;  // [pixels][parts][rank_pad], or null
  int store;     // its parts (kAdPlain and so on)
  int rank_pad;  // rank rounded up to 8
  int want_out;  // 0: only hidden
  int h_accs;    // accumulators that h's k-blocks alternate over
  void* out;     // NHWC, out_c channels
  int out_c;
  int map_h, map_w;  // fpn_adapter_split_kernel: the map behind the flattened one
  int bil_parts;     // 16-bit parts of the top-down weights on the tensor cores
};
constexpr int kAdMaxHAccs = 4;
int ad_h_accs(int num_kb) { return std::min(kAdMaxHAccs, (num_kb + 7) / 8); }

__device__ __forceinline__ int ad_adapter(const AdArgs& a, int n) {
  const int i = __ldg(a.index + n);
  return i >= 0 && i < a.adapters ? i : -1;
}

// v ~ the sum of its parts.  (A value beyond the type's range keeps the rest in the next part; infinity, and
// what exceeds the parts' ranges together, ends in the last one.)
template <typename T>
__device__ __forceinline__ float ad_clamp(float v) {
  constexpr float kMax = TcElem<T>::kFmt == 0 ? 65504.f : 3.3895313892515355e38f;
  return v > kMax ? kMax : (v < -kMax ? -kMax : v);
}
template <typename T>
__device__ __forceinline__ void ad_split(float v, uint16_t (&part)[kAdParts<T>]) {
#pragma unroll
  for (int i = 0; i < kAdParts<T>; ++i) {
    float c = v;
    if (i + 1 < kAdParts<T>) c = ad_clamp<T>(v);
    part[i] = Pack<T>::bits(c);
    v -= Pack<T>::unpack(static_cast<uint32_t>(part[i])).x;
  }
}

// What `hidden` holds.  fp16: two plain parts; h in three, the third for the bits below the second's steps
// (0 where that is normal, so that h stays the sum of the parts elsewhere); or dh in three.
enum : int { kAdPlain = 0, kAdFineH = 1, kAdFineDh = 2 };
template <typename T>
__host__ __device__ constexpr int ad_stored(int store) {
  return kAdParts<T> == kAdStored || store != kAdPlain ? kAdStored : 2;
}
// What a part of the fp16 forms is multiplied by.  dh is halved: values up to 131 008, as two plain parts
// take them.
__host__ __device__ constexpr float ad_factor(int store, int part) {
  if (store == kAdFineDh) return part == 0 ? 0x1p-1f : part == 1 ? 0x1p10f : 0x1p22f;
  return store == kAdFineH && part == 2 ? 0x1p11f : 1.f;
}
__host__ __device__ constexpr float ad_weight(int store, int part) { return 1.f / ad_factor(store, part); }

// Part i of v in `hidden`, taken off v.  (fp16: infinity and what exceeds the first two parts' ranges end
// in the second.)
template <typename T>
__device__ __forceinline__ uint32_t ad_take(float& v, int store, int i) {
  float c = v;
  if constexpr (kAdParts<T> == kAdStored) {
    if (i + 1 < kAdStored) c = ad_clamp<T>(v);
  } else {
    c = v * ad_factor(store, i);
    if (i == 0) {
      c = ad_clamp<T>(c);
      // (No subnormal first part of dh: the tensor cores align a step's products to the largest exponent
      // and count a subnormal's as 2^-14, which cost ddown 3e-6 at dh = 1.5e-7 where the second part alone
      // carries it to 5e-7.)
      if (store == kAdFineDh && fabsf(c) < 0x1p-14f) c = 0.f;
    }
  }
  const uint32_t bits = Pack<T>::bits(c);
  const float taken = Pack<T>::unpack(bits).x;
  if constexpr (kAdParts<T> == kAdStored) {
    v -= taken;
  } else {
    v = fmaf(-taken, ad_weight(store, i), v);  // (exact)
    if (i == 1 && !(fabsf(taken) < (store == kAdFineDh ? HUGE_VALF : 0x1p-14f))) v = 0.f;
  }
  return bits;
}

// The parts of eight values.  (A call: inlined, its registers were spilled in calls without `hidden` too, which
// cost these up to 5 %.)
template <typename T>
__device__ __noinline__ void ad_take8(uint4* dst, int stride, int store, float v0, float v1, float v2, float v3, float v4,
                                      float v5, float v6, float v7) {
  float v[8] = {v0, v1, v2, v3, v4, v5, v6, v7};
#pragma unroll
  for (int part = 0; part < kAdStored; ++part) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = ad_take<T>(v[2 * i], store, part);
      w[i] |= ad_take<T>(v[2 * i + 1], store, part) << 16;
    }
    if (part < ad_stored<T>(store)) dst[part * stride] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The taps of a pixel; one of weight 0 is another of the same pixel, so that what it holds stays out.
__device__ __forceinline__ TcTaps ad_taps(int py, int px, int H, int W, int Hc, int Wc, float scale_y, float scale_x) {
  TcTaps t = tc_taps(py, px, H, W, Hc, Wc, scale_y, scale_x);
  if (t.w01 == 0.f) t.xb = t.xa;
  if (t.w10 == 0.f) t.yb = t.ya;
  return t;
}

// kTaps: the top-down taps are added from global memory in the epilogue (their box exceeds 64 pixels).  Else
// an MMA adds them, which multiplies every pixel of the tile's coarse box by a weight, 0 for most: an
// infinity or a NaN reaches all 128 pixels of the tile.  So a block that has stored any such value (each warp
// looks at four of its pixels) computes its tiles once more with the taps that each pixel uses, from global
// memory.  (Taking them out of the box before the MMA, by the epilogue's idle warps, kept it waiting: 149
// instead of 144 us on P2 of eight images, which it takes without any of this.)
template <typename T, int RP, bool kTaps>
__global__ void __launch_bounds__(kAdThreads, 1)
    fpn_adapter_kernel(const __grid_constant__ CUtensorMap map_a,
                       const __grid_constant__ CUtensorMap map_b,
                       const __grid_constant__ CUtensorMap map_coarse,
                       const __grid_constant__ CUtensorMap map_u, const TcGemmArgs args,
                       const AdArgs ad) {
  constexpr int kParts = kAdParts<T>;
  using Cfg = AdCfg<RP, kParts, kTaps>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBars);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + S;
  uint64_t* accf_bar = bars + 2 * S;   // out accumulator final
  uint64_t* acce_bar = accf_bar + 1;   // ... and read
  uint64_t* hfull_bar = accf_bar + 2;  // h accumulator final
  uint64_t* tfull_bar = accf_bar + 3;  // h and up in shared memory
  uint64_t* wfull_bar = accf_bar + 4;  // the top-down weights in shared memory
  uint64_t* done_bar = accf_bar + 5;
  uint64_t* once_bar = accf_bar + 6;  // every tile stored once
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accf_bar + 7);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* nonfinite = abort_flag + 1;  // ... with an infinity or a NaN among them

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const bool bil_mma = !kTaps && args.coarse != nullptr;
  // Whether the block's tiles are computed again; a false after a timeout.
  auto again = [&]() {
    mbar_arrive(once_bar);
    return mbar_wait(once_bar, 0, abort_flag, args.status, kDevTimeoutAdapter) && *nonfinite != 0;
  };
  constexpr uint32_t kHCol = kTcBlockN;  // h accumulators: TMEM columns from 256, RP each

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(accf_bar, 1);
    mbar_init(acce_bar, 32 * kAdEpiWarps);
    mbar_init(hfull_bar, 1);
    mbar_init(tfull_bar, kAdEpiWarps * 32);
    mbar_init(wfull_bar, kTcBlockM * ad.bil_parts);
    mbar_init(done_bar, 1);
    mbar_init(once_bar, 32 + 1 + 32 * kAdEpiWarps);  // TMA warp, MMA issuer, epilogue
    *abort_flag = 0;
    *nonfinite = 0;
    fence_barrier_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
    prefetch_tmap(&map_u);
    if (bil_mma) prefetch_tmap(&map_coarse);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTcTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (whole warp)
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t box_bytes = static_cast<uint32_t>(args.cbox_w * args.cbox_h * 128);  // 64 channels
    for (bool bil = bil_mma;; bil = false) {
      const int nkb = args.num_kb + (bil ? 1 : 0);  // k-blocks of a tile: the products', the top-down add's
      for (int tile = blockIdx.x; ok && tile < args.num_tiles; tile += gridDim.x) {
        int n, x0, y0, slice;
        tc_tile_origin(args, tile, n, x0, y0, slice);
        const int adapter = ad_adapter(ad, n);
        if (!ad.want_out && adapter < 0) continue;
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, args.status, kDevTimeoutAdapter);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          uint8_t* const sa = smem + stage * Cfg::kStage;
          uint8_t* const su = sa + Cfg::kOffU;
          if (kb < args.num_kb) {
            if (lane == 0) {
              mbar_arrive_expect_tx(&full_bar[stage], kTcAStage + (ad.want_out ? kTcBStage : 0) +
                                                          (adapter >= 0 ? Cfg::kU : 0));
              tma_load_4d(sa, &map_a, &full_bar[stage], kb * 64, x0, y0, n, kPolicyEvictFirst);
              if (ad.want_out)
                tma_load_2d(sa + kTcAStage, &map_b, &full_bar[stage], kb * 64, slice * kTcBlockN,
                            kPolicyEvictLast);
              if (adapter >= 0)
                tma_load_4d(su, &map_u, &full_bar[stage], kb * 64, 0, 0, adapter, kPolicyEvictLast);
            }
          } else {
            // top-down k-block: the tile's coarse box as the B operand (the weights: the epilogue)
            uint8_t* const sb = sa + kTcAStage;
            tc_zero_btail(sb, lane, args.cbox_w * args.cbox_h, 4);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              const int cy = static_cast<int>(tc_src(y0, args.scale_y, args.Hc));
              const int cx = static_cast<int>(tc_src(x0, args.scale_x, args.Wc));
              mbar_arrive_expect_tx(&full_bar[stage], box_bytes * 4);
              for (int b = 0; b < 4; ++b)
                tma_load_4d(sb + b * (kTcCoarseMaxPix * 128), &map_coarse, &full_bar[stage], b * 64, cx,
                            cy, n, kPolicyEvictLast);
            }
          }
          ++issued;
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!bil) break;
      griddep_launch_dependents();
      if (!ok || !__all_sync(0xffffffffu, again())) break;
    }
    griddep_launch_dependents();
    if (lane == 0) {  // (matters only when another role gave up early)
      for (int i = 0; i < S && i < issued; ++i) {
        if (--stage < 0) {
          stage = S - 1;
          phase ^= 1u;
        }
        mbar_wait_drain(&full_bar[stage], phase);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t kFmt = TcElem<T>::kFmt;
      constexpr uint32_t idesc = make_idesc(kTcBlockM, kTcBlockN, kFmt, kFmt);
      constexpr uint32_t idesc_u = make_idesc(kTcBlockM, RP, kFmt, kFmt);
      constexpr uint32_t idesc_bmn = make_idesc(kTcBlockM, kTcBlockN, kFmt, kFmt, 1u);
      int stage = 0;
      uint32_t phase = 0, tile_phase = 0, h_phase = 0;
      const uint32_t t_addr = smem_u32(smem + Cfg::kOffT);
      bool ok = true;
      for (bool bil = bil_mma;; bil = false) {
        const int nkb = args.num_kb + (bil ? 1 : 0);
        for (int tile = blockIdx.x; ok && tile < args.num_tiles; tile += gridDim.x) {
          int n, x0, y0, slice;
          tc_tile_origin(args, tile, n, x0, y0, slice);
          const bool has = ad_adapter(ad, n) >= 0;
          if (!ad.want_out && !has) continue;
          if (!(ok = mbar_wait(acce_bar, tile_phase ^ 1u, abort_flag, args.status, kDevTimeoutAdapter))) break;
          tc_fence_after();
          int hset = 0;  // kb modulo h_accs
          for (int kb = 0; kb < nkb; ++kb) {
            if (!mbar_wait(&full_bar[stage], phase, abort_flag, args.status, kDevTimeoutAdapter)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = smem_u32(smem + stage * Cfg::kStage);
            const uint64_t adesc = sdesc_kmajor_sw128(sa);
            if (kb < args.num_kb) {
              const uint64_t bdesc = sdesc_kmajor_sw128(sa + kTcAStage);
              const uint64_t udesc = sdesc_kmajor_sw128(sa + Cfg::kOffU);
              // (the two products' steps alternate: the small ones, each waiting for the one before on its
              // accumulator, run behind the large ones)
              const uint32_t hacc = tmem_base + kHCol + static_cast<uint32_t>(hset * RP);
              const bool h_more = kb >= ad.h_accs;
              if (++hset == ad.h_accs) hset = 0;
#pragma unroll
              for (int k = 0; k < kMmaPerKb; ++k) {
                if (ad.want_out)
                  tc_mma_f16(tmem_base, adesc + 2u * k, bdesc + 2u * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
                if (has) tc_mma_f16(hacc, adesc + 2u * k, udesc + 2u * k, idesc_u, (h_more || k > 0) ? 1u : 0u);
              }
            } else {
              if (!mbar_wait(wfull_bar, tile_phase, abort_flag, args.status, kDevTimeoutAdapter)) {
                ok = false;
                break;
              }
              tc_fence_after();
              const uint64_t bdesc = sdesc_mnmajor_sw128(sa + kTcAStage, kTcCoarseMaxPix * 128);
              for (int part = 0; part < ad.bil_parts; ++part) {
                const uint64_t wdesc = sdesc_kmajor_sw128(t_addr + part * kTcAStage);
#pragma unroll
                for (int k = 0; k < kMmaPerKb; ++k)
                  tc_mma_f16(tmem_base, wdesc + 2u * k, bdesc + 128u * k, idesc_bmn, 1u);
              }
            }
            tc_commit(&empty_bar[stage]);
            if (++stage == S) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          if (has) {
            tc_commit(hfull_bar);
            if (ad.want_out) {
              if (!(ok = mbar_wait(tfull_bar, h_phase, abort_flag, args.status, kDevTimeoutAdapter))) break;
              tc_fence_after();
              const uint64_t vdesc = sdesc_kmajor_rows<Cfg::kRow>(smem_u32(smem + Cfg::kOffV));
#pragma unroll
              for (int part = 0; part < kParts; ++part) {
                const uint64_t tdesc = sdesc_kmajor_rows<Cfg::kRow>(t_addr + part * Cfg::kPart);
#pragma unroll
                for (int k = 0; k < RP / 16; ++k)
                  tc_mma_f16(tmem_base, tdesc + 2u * k, vdesc + 2u * k, idesc, 1u);
              }
            }
            h_phase ^= 1u;
          }
          if (ad.want_out) tc_commit(accf_bar);
          tile_phase ^= 1u;
        }
        if (!bil || !ok || !again()) break;
      }
      tc_commit(done_bar);
      mbar_wait_drain(done_bar, 0);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - 2;
    const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31
    const int cq = ew >> 2;        // output channels 64 * cq .. + 63
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_addr = smem_u32(smem + Cfg::kOffT), v_addr = smem_u32(smem + Cfg::kOffV);
    const uint32_t stage_addr = smem_u32(smem + Cfg::kOffStaging + ew * Cfg::kStaging);
    float* const bias_s = reinterpret_cast<float*>(smem + Cfg::kOffBias) + cq * kAdWarpCols;
    const int tw_shift = 31 - __clz(args.tile_w), tw_mask = args.tile_w - 1;  // (a power of two)
    uint32_t tile_phase = 0, h_phase = 0;
    int v_adapter = -1, v_slice = -1;  // what the up region holds
    // (each of the four warps writes the same values; with channel slices there is no bias)
    for (int i = lane; i < kAdWarpCols; i += 32)
      bias_s[i] = args.bias != nullptr ? __ldg(args.bias + cq * kAdWarpCols + i) : 0.f;
    __syncwarp();
    for (bool bil = bil_mma;; bil = false) {
      for (int tile = blockIdx.x; tile < args.num_tiles; tile += gridDim.x) {
        int n, x0, y0, slice;
        tc_tile_origin(args, tile, n, x0, y0, slice);
        const int adapter = ad_adapter(ad, n);
        const bool has = adapter >= 0;
        const int py = y0 + (row >> tw_shift), px = x0 + (row & tw_mask);
        const bool valid = py < args.H && px < args.W;
        // Here the tile before is through: its MMAs have read h, up and the top-down weights.
        if (bil && cq < ad.bil_parts) {
          // this pixel's row of the top-down weights, part cq: four of 64 coarse pixels
          const uint32_t wrow = t_addr + cq * kTcAStage + row * 128;
          const uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int j = 0; j < 8; ++j) st_shared_v4(wrow + ((j ^ (row & 7)) << 4), z);
          const TcTaps tp = tc_taps(py, px, args.H, args.W, args.Hc, args.Wc, args.scale_y, args.scale_x);
          const int cy0 = static_cast<int>(tc_src(y0, args.scale_y, args.Hc));
          const int cx0 = static_cast<int>(tc_src(x0, args.scale_x, args.Wc));
          int k[4] = {(tp.ya - cy0) * args.cbox_w + tp.xa - cx0, (tp.ya - cy0) * args.cbox_w + tp.xb - cx0,
                      (tp.yb - cy0) * args.cbox_w + tp.xa - cx0, (tp.yb - cy0) * args.cbox_w + tp.xb - cx0};
          float w[4] = {tp.w00, tp.w01, tp.w10, tp.w11};
          // (corners that coincide at the map's border add their weights)
#pragma unroll
          for (int i = 1; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < i; ++j)
              if (k[i] == k[j] && w[j] != 0.f) {
                w[j] += w[i];
                w[i] = 0.f;
              }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (w[i] == 0.f || k[i] < 0 || k[i] >= args.cbox_w * args.cbox_h) continue;
            const uint32_t byte = static_cast<uint32_t>(k[i]) * 2u;
            uint16_t bits = Pack<T>::bits(w[i]);
            if (cq > 0) bits = Pack<T>::bits(w[i] - Pack<T>::unpack(static_cast<uint32_t>(bits)).x);
            st_shared_u16(wrow + ((((byte >> 4) ^ (row & 7)) & 7) << 4) + (byte & 15), bits);
          }
          fence_proxy_async_smem();
          mbar_arrive(wfull_bar);
        }
        uint4* hid = nullptr;  // this thread's pixel of `hidden`
        if (ad.hidden != nullptr && slice == 0 && valid)
          hid = reinterpret_cast<uint4*>(
              static_cast<uint8_t*>(ad.hidden) +
              ((static_cast<size_t>(n) * args.H + py) * args.W + px) * ad.rank_pad * (2 * ad_stored<T>(ad.store)));
        if (has) {
          if (ad.want_out && cq >= 2 && (adapter != v_adapter || slice != v_slice)) {
            // up[a] (this slice's 256 rows): one row a thread of the upper two quarters
            const int c = (cq - 2) * kTcBlockM + row;
            const int ch = slice * kTcBlockN + c;
            const uint16_t* src = static_cast<const uint16_t*>(ad.v) + adapter * ad.va + ch * ad.vc;
#pragma unroll
            for (int j = 0; j < RP / 8; ++j) {
              uint4 q = make_uint4(0u, 0u, 0u, 0u);
              if (ch < ad.v_rows && j * 8 < ad.rank) {
                if (ad.v_vec) {
                  q = __ldg(reinterpret_cast<const uint4*>(src) + j);
                } else {
                  uint32_t w[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const int r = j * 8 + 2 * i;
                    const uint32_t lo = r < ad.rank ? __ldg(src + r * ad.vr) : 0;
                    const uint32_t hi = r + 1 < ad.rank ? __ldg(src + (r + 1) * ad.vr) : 0;
                    w[i] = lo | (hi << 16);
                  }
                  q = make_uint4(w[0], w[1], w[2], w[3]);
                }
              }
              st_shared_v4(v_addr + row_chunk<Cfg::kRow>(c, j), q);
            }
          }
          v_adapter = adapter;
          v_slice = slice;
          const float s = ad.scale * (ad.scales != nullptr ? __ldg(ad.scales + adapter) : 1.f);
          // (every warp waits for the tile's h, so that none runs ahead on the barriers below)
          const bool ok = mbar_wait(hfull_bar, h_phase, abort_flag, args.status, kDevTimeoutAdapter);
          if (!__all_sync(0xffffffffu, ok)) break;
          tc_fence_after();
          const uint32_t hacc = tmem_base + kHCol + lane_addr;
          // 8 columns at a time, by the quarters in turn
#pragma unroll 1
          for (int j = cq; j < RP / 8; j += 4) {
            uint32_t r[8];
            float h[8];
            __syncwarp();
            tmem_ld8(hacc + j * 8, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = __uint_as_float(r[i]);
            for (int q = 1; q < ad.h_accs; ++q) {
              tmem_ld8(hacc + q * RP + j * 8, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i) h[i] += __uint_as_float(r[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = j * 8 + i < ad.rank ? s * h[i] : 0.f;
            if (kParts == kAdStored || ad.want_out) {
              uint32_t w[kParts][4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint16_t p0[kParts], p1[kParts];
                ad_split<T>(h[2 * i], p0);
                ad_split<T>(h[2 * i + 1], p1);
#pragma unroll
                for (int part = 0; part < kParts; ++part)
                  w[part][i] = p0[part] | (static_cast<uint32_t>(p1[part]) << 16);
              }
#pragma unroll
              for (int part = 0; part < kParts; ++part) {
                const uint4 q = make_uint4(w[part][0], w[part][1], w[part][2], w[part][3]);
                if (ad.want_out) st_shared_v4(t_addr + part * Cfg::kPart + row_chunk<Cfg::kRow>(row, j), q);
                if (kParts == kAdStored && hid != nullptr && j * 8 < ad.rank_pad)
                  hid[(part * ad.rank_pad >> 3) + j] = q;
              }
            }
            if (kParts != kAdStored && hid != nullptr && j * 8 < ad.rank_pad)
              ad_take8<T>(hid + j, ad.rank_pad >> 3, ad.store, h[0], h[1], h[2], h[3], h[4], h[5], h[6], h[7]);
          }
          fence_proxy_async_smem();
          tc_fence_before();
          mbar_arrive(tfull_bar);
          h_phase ^= 1u;
          if (!ad.want_out) mbar_arrive(acce_bar);
        } else if (hid != nullptr && cq == 0) {
          for (int j = 0; j < ad.rank_pad * ad_stored<T>(ad.store) / 8; ++j) hid[j] = make_uint4(0u, 0u, 0u, 0u);
        }
        if (!ad.want_out) continue;

        const bool ok = mbar_wait(accf_bar, tile_phase, abort_flag, args.status, kDevTimeoutAdapter);
        if (!__all_sync(0xffffffffu, ok)) break;
        tile_phase ^= 1u;
        tc_fence_after();
        if (!kTaps && bil_mma && !bil) {  // once more, with the taps
          const TcTaps tp = ad_taps(py, px, args.H, args.W, args.Hc, args.Wc, args.scale_y, args.scale_x);
          const T* c = static_cast<const T*>(args.coarse) +
                       static_cast<size_t>(n) * args.Hc * args.Wc * kTcBlockN + cq * kAdWarpCols;
          T* const o = static_cast<T*>(ad.out) +
                       ((static_cast<size_t>(n) * args.H + py) * args.W + px) * kTcBlockN + cq * kAdWarpCols;
#pragma unroll 1
          for (int j = 0; j < kAdWarpCols / 8; ++j) {
            uint32_t r[8];
            __syncwarp();
            tmem_ld8(tmem_base + cq * kAdWarpCols + j * 8 + lane_addr, r);
            tmem_wait_ld();
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]) + bias_s[j * 8 + i];
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
              const float wk = k == 0 ? tp.w00 : k == 1 ? tp.w01 : k == 2 ? tp.w10 : tp.w11;
              const size_t at = static_cast<size_t>(k < 2 ? tp.ya : tp.yb) * args.Wc + ((k & 1) == 0 ? tp.xa : tp.xb);
              const uint4 q = __ldg(reinterpret_cast<const uint4*>(c + at * kTcBlockN) + j);
              const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = Pack<T>::unpack(u[e]);
                v[2 * e] = fmaf(wk, f.x, v[2 * e]);
                v[2 * e + 1] = fmaf(wk, f.y, v[2 * e + 1]);
              }
            }
            if (valid)
              reinterpret_cast<uint4*>(o)[j] = make_uint4(Pack<T>::pack(v[0], v[1]), Pack<T>::pack(v[2], v[3]),
                                                          Pack<T>::pack(v[4], v[5]), Pack<T>::pack(v[6], v[7]));
          }
          tc_fence_before();
          mbar_arrive(acce_bar);
          continue;
        }
        // The warp's accumulators go to registers at once, so that the next tile's MMAs start while
        // they are converted and stored.
        uint32_t rr[kAdWarpCols];
        __syncwarp();
#pragma unroll
        for (int q = 0; q < kAdWarpCols / 32; ++q)
          tmem_ld32(tmem_base + cq * kAdWarpCols + q * 32 + lane_addr,
                    *reinterpret_cast<uint32_t(*)[32]>(&rr[q * 32]));
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive(acce_bar);

        TcTaps tp{};
        const T* tap[4];
        if constexpr (kTaps) {
          tp = ad_taps(py, px, args.H, args.W, args.Hc, args.Wc, args.scale_y, args.scale_x);
          const T* c = static_cast<const T*>(args.coarse) +
                       static_cast<size_t>(n) * args.Hc * args.Wc * kTcBlockN + cq * kAdWarpCols;
          tap[0] = c + (static_cast<size_t>(tp.ya) * args.Wc + tp.xa) * kTcBlockN;
          tap[1] = c + (static_cast<size_t>(tp.ya) * args.Wc + tp.xb) * kTcBlockN;
          tap[2] = c + (static_cast<size_t>(tp.yb) * args.Wc + tp.xa) * kTcBlockN;
          tap[3] = c + (static_cast<size_t>(tp.yb) * args.Wc + tp.xb) * kTcBlockN;
        }
        uint4 pk[kAdWarpCols / 8];  // the pixel's channels, rounded
#pragma unroll
        for (int step = 0; step < kAdWarpCols / 16; ++step) {
          float v[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 b = *reinterpret_cast<const float4*>(bias_s + step * 16 + 4 * i);
            v[4 * i + 0] = __uint_as_float(rr[step * 16 + 4 * i + 0]) + b.x;
            v[4 * i + 1] = __uint_as_float(rr[step * 16 + 4 * i + 1]) + b.y;
            v[4 * i + 2] = __uint_as_float(rr[step * 16 + 4 * i + 2]) + b.z;
            v[4 * i + 3] = __uint_as_float(rr[step * 16 + 4 * i + 3]) + b.w;
          }
          if constexpr (kTaps) {
            const float w[4] = {tp.w00, tp.w01, tp.w10, tp.w11};
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint4 q = __ldg(reinterpret_cast<const uint4*>(tap[k] + step * 16) + h);
                const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 f = Pack<T>::unpack(u[e]);
                  v[8 * h + 2 * e] = fmaf(w[k], f.x, v[8 * h + 2 * e]);
                  v[8 * h + 2 * e + 1] = fmaf(w[k], f.y, v[8 * h + 2 * e + 1]);
                }
              }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
            pk[2 * step + h] =
                make_uint4(Pack<T>::pack(v[8 * h + 0], v[8 * h + 1]), Pack<T>::pack(v[8 * h + 2], v[8 * h + 3]),
                           Pack<T>::pack(v[8 * h + 4], v[8 * h + 5]), Pack<T>::pack(v[8 * h + 6], v[8 * h + 7]));
        }
        // 8 pixels at a time through the warp's 1 KB of shared memory, so that 8 lanes write the 128 bytes of a
        // pixel: lane l stores chunk l % 8 of pixels l / 8 and l / 8 + 4.  (32 pixels of 16 channels at a time
        // touched 16 lines an instruction instead of 4: 145 us for P2 of eight images.)
        const int scol = slice * kTcBlockN + cq * kAdWarpCols + (lane & 7) * 8;
        const bool in_cols = scol < ad.out_c;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if ((lane >> 3) == g) {
#pragma unroll
            for (int j = 0; j < 8; ++j) st_shared_v4(stage_addr + row_chunk<128>(lane & 7, j), pk[j]);
          }
          __syncwarp();
          uint4 o[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) o[i] = ld_shared_v4(stage_addr + row_chunk<128>((lane >> 3) + 4 * i, lane & 7));
          __syncwarp();
          if (g == 0 && bil) {  // (all 64 channels, of four pixels)
            constexpr uint32_t kInf = TcElem<T>::kFmt == 0 ? 0x7c007c00u : 0x7f807f80u, kAbs = 0x7fff7fffu;
            const uint32_t most = __vmaxu2(__vmaxu2(o[0].x & kAbs, o[0].y & kAbs), __vmaxu2(o[0].z & kAbs, o[0].w & kAbs));
            if (__vcmpgeu2(most, kInf) != 0u) *nonfinite = 1;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = quarter * 32 + g * 8 + (lane >> 3) + 4 * i;
            const int sy = y0 + (r >> tw_shift), sx = x0 + (r & tw_mask);
            if (in_cols && sy < args.H && sx < args.W)
              *reinterpret_cast<uint4*>(static_cast<T*>(ad.out) +
                                        ((static_cast<size_t>(n) * args.H + sy) * args.W + sx) * ad.out_c + scol) = o[i];
          }
        }
      }
      if (!bil || !__all_sync(0xffffffffu, again())) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, kTcTmemCols);
  }
}

// ------------------------------------------------------------------ few tiles
// The same forward where a map has few tiles: a cluster of S CTAs shares a tile, each with 1 / S of the
// k-blocks: one CTA needs 0.4 us for a k-block, most of it the tensor cores on 128 rows whatever the
// map fills of them.  h up[a]^T is linear in h, so each CTA adds the share of its own partial h to its partial
// product on the tensor cores; then all put their fp32 partial products into their own shared memory,
// and after a cluster barrier CTA r reads rows r, r + S, .. of all S, adds them in order with the bias and
// the top-down taps (fetched while the k-loop runs), and stores those rows.
// Shared memory: the ring, up[a], barriers; after the k-loop the ring holds the parts of h, then the partial
// product, and the partial h.
struct AsSmem {
  int stages, stage, up, h, bars, total;
};
__host__ __device__ constexpr AsSmem as_smem(int rp) {
  AsSmem m{};
  m.stages = rp <= 32 ? 4 : 3;
  m.stage = kTcAStage + kTcBStage + rp * 128;
  m.up = m.stages * m.stage;
  m.h = kTcBlockM * kTcBlockN * 4;
  m.bars = m.up + kTcBlockN * rp * 2;
  m.total = m.bars + 256 + 1024;
  return m;
}
constexpr bool as_smem_fits(int rp) {
  return as_smem(rp).total <= 232448 && as_smem(rp).h + kTcBlockM * rp * 4 <= as_smem(rp).up;
}
static_assert(as_smem_fits(16) && as_smem_fits(32) && as_smem_fits(64), "adapter split smem");

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}
// (zeros without `on`; no branch, so that a thread's loads stay together)
__device__ __forceinline__ float4 ld_cluster_f4_if(bool on, uint32_t addr) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "@p ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "+f"(v.x), "+f"(v.y), "+f"(v.z), "+f"(v.w)
      : "r"(addr), "r"(static_cast<int>(on)));
  return v;
}
__device__ __forceinline__ void st_shared_f4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

template <typename T, int RP, int S>
__global__ void __launch_bounds__(kAdThreads, 1)
    fpn_adapter_split_kernel(const __grid_constant__ CUtensorMap map_a,
                             const __grid_constant__ CUtensorMap map_b,
                             const __grid_constant__ CUtensorMap map_u, const TcGemmArgs args,
                             const AdArgs ad) {
  constexpr int kParts = kAdParts<T>;
  constexpr int kOwn = kTcBlockM / S;  // rows that this CTA finishes
  constexpr int kRows = kOwn / 8;      // ... of a thread
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  constexpr AsSmem lay = as_smem(RP);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + lay.bars);
  uint64_t* empty_bar = full_bar + 4;
  uint64_t* accf_bar = full_bar + 8;   // partial product final
  uint64_t* hfull_bar = full_bar + 9;  // partial h final
  uint64_t* tfull_bar = full_bar + 10;  // h and up in shared memory
  uint64_t* done_bar = full_bar + 11;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full_bar + 12);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  if (threadIdx.x == 0) {
    for (int s = 0; s < lay.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(accf_bar, 1);
    mbar_init(hfull_bar, 1);
    mbar_init(tfull_bar, 32 * kAdEpiWarps);
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
    prefetch_tmap(&map_u);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTcTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();

  int n, x0, y0;  // (a map of one row: pixels x0 .. x0 + 127 of image n)
  tc_tile_origin(args, static_cast<int>(blockIdx.x) / S, n, x0, y0);
  const int adapter = ad_adapter(ad, n);
  const bool has = adapter >= 0;
  const int kb0 = rank * args.num_kb / S, kb1 = (rank + 1) * args.num_kb / S;  // non-empty (host)
  const uint32_t base = smem_u32(smem);

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, args.status, kDevTimeoutAdapter)) break;
        uint8_t* const sa = smem + stage * lay.stage;
        mbar_arrive_expect_tx(&full_bar[stage], kTcAStage + kTcBStage + (has ? RP * 128 : 0));
        tma_load_4d(sa, &map_a, &full_bar[stage], kb * 64, x0, 0, n, kPolicyEvictFirst);
        tma_load_2d(sa + kTcAStage, &map_b, &full_bar[stage], kb * 64, 0, kPolicyEvictLast);
        if (has)
          tma_load_4d(sa + kTcAStage + kTcBStage, &map_u, &full_bar[stage], kb * 64, 0, 0, adapter,
                      kPolicyEvictLast);
        ++issued;
        if (++stage == lay.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      for (int i = 0; i < lay.stages && i < issued; ++i) {  // (matters only when another role gave up)
        if (--stage < 0) {
          stage = lay.stages - 1;
          phase ^= 1u;
        }
        mbar_wait_drain(&full_bar[stage], phase);
      }
    }
    __syncwarp();
    griddep_launch_dependents();
    cluster_sync_all();
    cluster_arrive();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t kFmt = TcElem<T>::kFmt;
      constexpr uint32_t idesc = make_idesc(kTcBlockM, kTcBlockN, kFmt, kFmt);
      constexpr uint32_t idesc_u = make_idesc(kTcBlockM, RP, kFmt, kFmt);
      int stage = 0, hset = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, abort_flag, args.status, kDevTimeoutAdapter)) break;
        tc_fence_after();
        const uint32_t sa = base + stage * lay.stage;
        const uint64_t adesc = sdesc_kmajor_sw128(sa);
        const uint64_t bdesc = sdesc_kmajor_sw128(sa + kTcAStage);
        const uint64_t udesc = sdesc_kmajor_sw128(sa + kTcAStage + kTcBStage);
        const uint32_t hacc = tmem_base + kTcBlockN + static_cast<uint32_t>(hset * RP);
        const bool h_more = kb - kb0 >= ad.h_accs;
        if (++hset == ad.h_accs) hset = 0;
#pragma unroll
        for (int k = 0; k < kMmaPerKb; ++k) {
          tc_mma_f16(tmem_base, adesc + 2u * k, bdesc + 2u * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
          if (has) tc_mma_f16(hacc, adesc + 2u * k, udesc + 2u * k, idesc_u, (h_more || k > 0) ? 1u : 0u);
        }
        tc_commit(&empty_bar[stage]);
        if (++stage == lay.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (has) {
        tc_commit(hfull_bar);
        if (mbar_wait(tfull_bar, 0, abort_flag, args.status, kDevTimeoutAdapter)) {
          tc_fence_after();
          const uint64_t vdesc = sdesc_kmajor_rows<RP * 2>(base + lay.up);
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            const uint64_t tdesc = sdesc_kmajor_rows<RP * 2>(base + part * (kTcBlockM * RP * 2));
#pragma unroll
            for (int k = 0; k < RP / 16; ++k)
              tc_mma_f16(tmem_base, tdesc + 2u * k, vdesc + 2u * k, idesc, 1u);
          }
        }
      }
      tc_commit(accf_bar);
      tc_commit(done_bar);
      mbar_wait_drain(done_bar, 0);
    }
    __syncwarp();
    cluster_sync_all();
    cluster_arrive();
  } else {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - 2;
    const int t = ew * 32 + lane;
    const int c4 = (t & 63) * 4;  // output channels c4 .. c4 + 3
    const int r0 = (t >> 6) * S + rank;  // own rows r0, r0 + 8 S, ..
    const int pixels = args.W;    // of an image
    if (has && t < kTcBlockN) {  // up[a], a row a thread
      const uint16_t* src = static_cast<const uint16_t*>(ad.v) + adapter * ad.va + t * ad.vc;
#pragma unroll
      for (int j = 0; j < RP / 8; ++j) {
        uint4 q = make_uint4(0u, 0u, 0u, 0u);
        if (j * 8 < ad.rank) {
          if (ad.v_vec) {
            q = __ldg(reinterpret_cast<const uint4*>(src) + j);
          } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = j * 8 + 2 * i;
              const uint32_t lo = r < ad.rank ? __ldg(src + r) : 0;
              const uint32_t hi = r + 1 < ad.rank ? __ldg(src + r + 1) : 0;
              w[i] = lo | (hi << 16);
            }
            q = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        st_shared_v4(base + lay.up + row_chunk<RP * 2>(t, j), q);
      }
    }
    // (rows past the map take its last pixel: their loads need no branch, and they are not stored)
    float4 v[kRows];
    {
      float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
      if (args.bias != nullptr) b = __ldg(reinterpret_cast<const float4*>(args.bias + c4));
#pragma unroll
      for (int i = 0; i < kRows; ++i) v[i] = b;
    }
    if (args.coarse != nullptr && x0 + r0 < pixels) {
      const T* coarse = static_cast<const T*>(args.coarse) +
                        static_cast<size_t>(n) * args.Hc * args.Wc * kTcBlockN + c4;
      constexpr int kBatch = kRows < 4 ? kRows : 4;
#pragma unroll
      for (int i0 = 0; i0 < kRows; i0 += kBatch) {
        uint2 q[kBatch][4];
        float w[kBatch][4];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int p = min(x0 + r0 + 8 * S * (i0 + i), pixels - 1);
          const int py = p / ad.map_w, px = p - py * ad.map_w;
          const TcTaps tp = ad_taps(py, px, ad.map_h, ad.map_w, args.Hc, args.Wc, args.scale_y, args.scale_x);
          const T* top = coarse + static_cast<size_t>(tp.ya) * args.Wc * kTcBlockN;
          const T* bottom = coarse + static_cast<size_t>(tp.yb) * args.Wc * kTcBlockN;
          q[i][0] = __ldg(reinterpret_cast<const uint2*>(top + tp.xa * kTcBlockN));
          q[i][1] = __ldg(reinterpret_cast<const uint2*>(top + tp.xb * kTcBlockN));
          q[i][2] = __ldg(reinterpret_cast<const uint2*>(bottom + tp.xa * kTcBlockN));
          q[i][3] = __ldg(reinterpret_cast<const uint2*>(bottom + tp.xb * kTcBlockN));
          w[i][0] = tp.w00;
          w[i][1] = tp.w01;
          w[i][2] = tp.w10;
          w[i][3] = tp.w11;
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 lo = Pack<T>::unpack(q[i][e].x), hi = Pack<T>::unpack(q[i][e].y);
            float4& o = v[i0 + i];
            o.x = fmaf(w[i][e], lo.x, o.x);
            o.y = fmaf(w[i][e], lo.y, o.y);
            o.z = fmaf(w[i][e], hi.x, o.z);
            o.w = fmaf(w[i][e], hi.y, o.w);
          }
      }
    }
    const float hs = has ? ad.scale * (ad.scales != nullptr ? __ldg(ad.scales + adapter) : 1.f) : 0.f;

    const int quarter = warp & 3, cq = ew >> 2;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    bool ok = true;
    if (has) {
      ok = mbar_wait(hfull_bar, 0, abort_flag, args.status, kDevTimeoutAdapter);
      if (__all_sync(0xffffffffu, ok)) {
        // The ring is free: the MMAs, and so the loads, are through.
        tc_fence_after();
#pragma unroll 1
        for (int j = cq; j < RP / 8; j += 4) {
          float h[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = 0.f;
          for (int a = 0; a < ad.h_accs; ++a) {
            uint32_t rr[8];
            tmem_ld8(tmem_base + kTcBlockN + lane_addr + a * RP + j * 8, rr);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] += __uint_as_float(rr[i]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = j * 8 + i < ad.rank ? hs * h[i] : 0.f;
          if (ad.hidden != nullptr) {
            const uint32_t dst = base + lay.h + (row * RP + j * 8) * 4;
            st_shared_f4(dst, h[0], h[1], h[2], h[3]);
            st_shared_f4(dst + 16, h[4], h[5], h[6], h[7]);
          }
          uint16_t p[8][kParts];
#pragma unroll
          for (int i = 0; i < 8; ++i) ad_split<T>(h[i], p[i]);
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = p[2 * i][part] | (static_cast<uint32_t>(p[2 * i + 1][part]) << 16);
            st_shared_v4(base + part * (kTcBlockM * RP * 2) + row_chunk<RP * 2>(row, j),
                         make_uint4(w[0], w[1], w[2], w[3]));
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
      }
      mbar_arrive(tfull_bar);
    }
    ok = mbar_wait(accf_bar, 0, abort_flag, args.status, kDevTimeoutAdapter);
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      if (x0 + quarter * 32 < pixels) {  // (rows past the map stay unwritten, and unread)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t rr[32];
          tmem_ld32(tmem_base + lane_addr + cq * 64 + q * 32, rr);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 8; ++j) {  // (16-byte chunk c of row r at c ^ (r % 8): no bank conflicts)
            const int chunk = cq * 16 + q * 8 + j;
            st_shared_v4(base + row * (kTcBlockN * 4) + ((chunk ^ (row & 7)) << 4),
                         make_uint4(rr[4 * j], rr[4 * j + 1], rr[4 * j + 2], rr[4 * j + 3]));
          }
        }
      }
      tc_fence_before();
    }
    __syncwarp();
    cluster_sync_all();

    uint32_t part[S];
#pragma unroll
    for (int s = 0; s < S; ++s) part[s] = mapa_shared(base, s);
    const bool rows = x0 + r0 < pixels;  // this warp has any
    if (rows) {
      float4 q[kRows][S];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int row = r0 + 8 * S * i;
        const uint32_t off = row * (kTcBlockN * 4) + (((c4 >> 2) ^ (row & 7)) << 4);
#pragma unroll
        for (int s = 0; s < S; ++s) q[i][s] = ld_cluster_f4_if(x0 + row < pixels, part[s] + off);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
#pragma unroll
        for (int s = 1; s < S; ++s) {
          q[i][0].x += q[i][s].x;
          q[i][0].y += q[i][s].y;
          q[i][0].z += q[i][s].z;
          q[i][0].w += q[i][s].w;
        }
        v[i].x += q[i][0].x;
        v[i].y += q[i][0].y;
        v[i].z += q[i][0].z;
        v[i].w += q[i][0].w;
      }
    }
    if (ad.hidden != nullptr) {
      // h of the own rows, four columns a thread, in its parts (zeros without an adapter)
      const int q4 = ad.rank_pad >> 2;
      for (int i = t; i < kOwn * q4; i += 32 * kAdEpiWarps) {
        const int own = i / q4 * S + rank, c = (i % q4) * 4;
        const int p = x0 + own;
        if (p >= pixels) break;  // (rows grow with i)
        float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
        if (has) {
#pragma unroll
          for (int s = 0; s < S; ++s) {
            const float4 q = ld_cluster_f4(part[s] + lay.h + (own * RP + c) * 4);
            h.x += q.x;
            h.y += q.y;
            h.z += q.z;
            h.w += q.w;
          }
        }
        uint16_t* hid = static_cast<uint16_t*>(ad.hidden) +
                        (static_cast<size_t>(n) * pixels + p) * ad.rank_pad * ad_stored<T>(ad.store) + c;
#pragma unroll
        for (int k = 0; k < kAdStored; ++k) {
          uint2 q;
          q.x = ad_take<T>(h.x, ad.store, k);
          q.x |= ad_take<T>(h.y, ad.store, k) << 16;
          q.y = ad_take<T>(h.z, ad.store, k);
          q.y |= ad_take<T>(h.w, ad.store, k) << 16;
          if (k < ad_stored<T>(ad.store)) *reinterpret_cast<uint2*>(hid + k * ad.rank_pad) = q;
        }
      }
    }
    __syncwarp();
    cluster_arrive();  // (the others' partials are read)
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int p = x0 + r0 + 8 * S * i;
      if (p >= pixels) break;
      *reinterpret_cast<uint2*>(static_cast<T*>(ad.out) + (static_cast<size_t>(n) * pixels + p) * kTcBlockN + c4) =
          make_uint2(Pack<T>::pack(v[i].x, v[i].y), Pack<T>::pack(v[i].z, v[i].w));
    }
  }

  tc_fence_before();
  __syncwarp();
  cluster_wait();  // (no CTA ends while another reads its partials)
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTcTmemCols);
  }
}

// ------------------------------------------------------------------ adapter gradients
// part[unit][r][c] = sum over the unit's pixels of h[p][r] q[p][c]: for the channel blocks of x with
// h = dh (ddown), and for dy with h (dup).  A tcgen05 GEMM over pixels (both operands MN-major
// 64-pixel boxes): M = 256 channels in two accumulators, N = parts x rank_pad columns, the parts of
// h side by side, weighed and added when the accumulators are read.  Where TMEM has room (N <= 128), the k-blocks
// alternate over two pairs of accumulators: at most 64 steps on one (see the rounding above).
constexpr int kAgChunk = 64 * 128;
constexpr int kAgStages = 4;
constexpr int kAgQ = 4 * kAgChunk;                 // 256 channels
constexpr int kAgStage = kAgQ + 3 * kAgChunk;      // + up to 192 columns of h
constexpr int kAgOffBars = kAgStages * kAgStage;
constexpr int kAgSmemBytes = kAgOffBars + 256 + 1024;
static_assert(kAgSmemBytes <= 232448, "adapter gradient smem");

struct AgArgs {
  const int* index;
  int adapters;
  int n0;                 // first image of the launch
  int splits, per, num_kb;  // 64-pixel k-blocks of an image: num_kb, `per` of them a split
  int blocks, x_blocks;     // 256-channel blocks: x_blocks of x, then one of dy
  int rank_pad;
  int store;  // of h (dh: kAdFineDh)
  float* part;  // [image - n0][split][block][rank_pad][256]
  int* status;
};

template <typename T>
__global__ void __launch_bounds__(kTcThreads, 1)
    fpn_adapter_grad_kernel(const __grid_constant__ CUtensorMap map_x,
                            const __grid_constant__ CUtensorMap map_dy,
                            const __grid_constant__ CUtensorMap map_dh,
                            const __grid_constant__ CUtensorMap map_h, const AgArgs a) {
  constexpr int S = kAgStages;
  int u = static_cast<int>(blockIdx.x);
  const int block = u % a.blocks;
  u /= a.blocks;
  const int split = u % a.splits;
  const int n = a.n0 + u / a.splits;
  const int adapter = __ldg(a.index + n);
  if (adapter < 0 || adapter >= a.adapters) {  // (before any barrier or TMEM)
    griddep_wait();
    return;
  }

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kAgOffBars);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + S;
  uint64_t* accf_bar = bars + 2 * S;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accf_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const bool is_x = block < a.x_blocks;
  const CUtensorMap* mq = is_x ? &map_x : &map_dy;
  const CUtensorMap* mh = is_x ? &map_dh : &map_h;
  const int c0 = is_x ? block * 256 : 0;
  const int kb0 = split * a.per, kb1 = min(a.num_kb, kb0 + a.per);  // non-empty (host)
  constexpr bool kPlain = kAdParts<T> == kAdStored;  // all parts count once
  const int store = is_x ? kAdFineDh : a.store;
  const int parts = ad_stored<T>(store);
  const int cols = (parts * a.rank_pad + 15) / 16 * 16;  // (columns past the parts are zeros)
  const int hchunks = (cols + 63) / 64;
  const int sets = cols <= 128 ? 2 : 1;  // accumulators at columns 256 * half + 128 * set

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(accf_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(mq);
    prefetch_tmap(mh);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, a.status, kDevTimeoutAdapter)) break;
        uint8_t* const sq = smem + stage * kAgStage;
        mbar_arrive_expect_tx(&full_bar[stage], kAgQ + hchunks * kAgChunk);
        for (int j = 0; j < 4; ++j)
          tma_load_4d(sq + j * kAgChunk, mq, &full_bar[stage], c0 + j * 64, kb * 64, 0, n,
                      kPolicyEvictFirst);
        for (int j = 0; j < hchunks; ++j)
          tma_load_4d(sq + kAgQ + j * kAgChunk, mh, &full_bar[stage], j * 64, kb * 64, 0, n,
                      kPolicyEvictLast);
        ++issued;
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
      griddep_launch_dependents();
      for (int i = 0; i < S && i < issued; ++i) {
        if (--stage < 0) {
          stage = S - 1;
          phase ^= 1u;
        }
        mbar_wait_drain(&full_bar[stage], phase);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc(kTcBlockM, cols, TcElem<T>::kFmt, TcElem<T>::kFmt, 1u, 1u);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, abort_flag, a.status, kDevTimeoutAdapter)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t q = smem_u32(smem + stage * kAgStage);
        const uint64_t a0 = sdesc_mnmajor_sw128(q, kAgChunk);
        const uint64_t a1 = sdesc_mnmajor_sw128(q + 2 * kAgChunk, kAgChunk);
        const uint64_t b = sdesc_mnmajor_sw128(q + kAgQ, kAgChunk);
#pragma unroll
        for (int k = 0; k < kMmaPerKb; ++k) {  // 16 pixels per step
          const uint32_t set = (kb - kb0) % sets, d = tmem_base + 128u * set;
          const uint32_t acc = (kb - kb0 >= sets || k > 0) ? 1u : 0u;
          tc_mma_f16(d, a0 + 128u * k, b + 128u * k, idesc, acc);
          tc_mma_f16(d + 256, a1 + 128u * k, b + 128u * k, idesc, acc);
        }
        tc_commit(&empty_bar[stage]);
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // (after a timeout: what was issued completes before TMEM goes, and the partial is unused)
      tc_commit(accf_bar);
      if (!ok) mbar_wait_drain(accf_bar, 0);
    }
  } else {
    const int ew = warp - 2, quarter = warp & 3, half = ew >> 2;
    const bool ok = mbar_wait(accf_bar, 0, abort_flag, a.status, kDevTimeoutAdapter);
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      const uint32_t acc = tmem_base + half * 256 + (static_cast<uint32_t>(quarter * 32) << 16);
      const int used = min(sets, kb1 - kb0);
      float* dst = a.part + ((static_cast<size_t>(n - a.n0) * a.splits + split) * a.blocks + block) *
                                a.rank_pad * 256 +
                   half * 128 + quarter * 32 + lane;
      for (int r = 0; r < a.rank_pad; r += 8) {
        float sum[8] = {};
#pragma unroll
        for (int part = kAdStored - 1; part >= 0; --part) {  // the smallest first
          if (part >= parts) continue;
          const float weight = kPlain ? 1.f : ad_weight(store, part);
          for (int set = 0; set < used; ++set) {
            uint32_t v[8];
            __syncwarp();
            tmem_ld8(acc + 128 * set + part * a.rank_pad + r, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] = fmaf(weight, __uint_as_float(v[i]), sum[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[(r + i) * 256] = sum[i];
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Adds an adapter's partials over its images (in order) and their splits.  Block (adapter,
// channel block, r); thread = channel.  `more`: adds to what the outputs hold.
struct ArArgs {
  const int* index;
  int n0, images, splits, blocks, x_blocks, rank, rank_pad, Cin;
  const float* part;
  float* ddown;  // [L][rank][Cin]
  float* dup;    // [L][256][rank]
  int more;
};
constexpr int kArList = 1024;
__global__ void __launch_bounds__(256) adapter_reduce_kernel(const ArArgs a) {
  __shared__ int list[kArList];
  __shared__ int count;
  const int r = blockIdx.x % a.rank, block = blockIdx.x / a.rank;
  const int adapter = blockIdx.y;
  const int c = threadIdx.x;
  griddep_wait();
  float acc = 0.f;
  for (int i0 = 0; i0 < a.images; i0 += kArList) {
    __syncthreads();
    if (threadIdx.x < 32) {  // the adapter's images among the next kArList, in order
      int k = 0;
      for (int i = i0; i < min(a.images, i0 + kArList); i += 32) {
        const int n = i + threadIdx.x;
        const bool hit = n < a.images && n < i0 + kArList && __ldg(a.index + a.n0 + n) == adapter;
        const unsigned m = __ballot_sync(0xffffffffu, hit);
        if (hit) list[k + __popc(m & ((1u << threadIdx.x) - 1u))] = n;
        k += __popc(m);
      }
      if (threadIdx.x == 0) count = k;
    }
    __syncthreads();
    const size_t step = static_cast<size_t>(a.blocks) * a.rank_pad * 256;
    for (int i = 0; i < count; ++i) {
      const float* p = a.part + static_cast<size_t>(list[i]) * a.splits * step +
                       (static_cast<size_t>(block) * a.rank_pad + r) * 256 + c;
#pragma unroll 4
      for (int s = 0; s < a.splits; ++s) acc += p[s * step];
    }
  }
  float* out;
  if (block < a.x_blocks) {
    if (block * 256 + c >= a.Cin) return;
    out = a.ddown + (static_cast<size_t>(adapter) * a.rank + r) * a.Cin + block * 256 + c;
  } else {
    out = a.dup + (static_cast<size_t>(adapter) * 256 + c) * a.rank + r;
  }
  *out = a.more ? *out + acc : acc;
}

// The backward's operands: up [L][256][R] -> [L][R][256] (block l), and W [256][K] -> [K rounded up to
// 256][256], 32 input channels a block, zeros past K.
__global__ void __launch_bounds__(256)
    adapter_transpose_kernel(const uint16_t* __restrict__ up, uint16_t* __restrict__ up_t, int rank, int adapters,
                             const uint16_t* __restrict__ w, uint16_t* __restrict__ w_t, int K) {
  griddep_launch_dependents();
  const int t = static_cast<int>(threadIdx.x);
  if (static_cast<int>(blockIdx.x) < adapters) {
    const size_t a = blockIdx.x;
#pragma unroll 4
    for (int r = 0; r < rank; ++r) up_t[(a * rank + r) * 256 + t] = __ldg(up + (a * 256 + t) * rank + r);
    return;
  }
  __shared__ __align__(16) uint16_t tile[32][256 + 8];
  const int k0 = (static_cast<int>(blockIdx.x) - adapters) * 32;
  uint4 q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 64 + (t >> 2), k = k0 + (t & 3) * 8;
    q[i] = k < K ? __ldg(reinterpret_cast<const uint4*>(w + static_cast<size_t>(row) * K + k)) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      tile[(t & 3) * 8 + e][i * 64 + (t >> 2)] = static_cast<uint16_t>(u[e >> 1] >> (16 * (e & 1)));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 8 + (t >> 5);
    *reinterpret_cast<uint4*>(w_t + static_cast<size_t>(k0 + row) * 256 + (t & 31) * 8) =
        *reinterpret_cast<const uint4*>(&tile[row][(t & 31) * 8]);
  }
}

// ------------------------------------------------------------------ host side
template <typename T, int RP, bool kTaps>
cudaError_t launch_adapter_rp(const TcPlan& p, const CUtensorMap& map_u, const AdArgs& ad, const LaunchOpts& opts,
                              cudaStream_t s) {
  using Cfg = AdCfg<RP, kAdParts<T>, kTaps>;
  auto kern = fpn_adapter_kernel<T, RP, kTaps>;
  static std::atomic<bool> configured[64];
  cudaError_t e = once_per_device(configured, [&] {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
  });
  if (e != cudaSuccess) return e;
  TcGemmArgs a;
  std::memcpy(&a, p.args, sizeof(a));
  return launch_ex(kern, dim3(p.grid), dim3(kAdThreads), Cfg::kSmemBytes, s, opts, 1, p.map_a,
                   p.map_b, p.map_coarse, map_u, a, ad);
}
template <typename T, bool kTaps>
cudaError_t launch_adapter_rank(const TcPlan& p, const CUtensorMap& map_u, const AdArgs& ad, const LaunchOpts& opts,
                                cudaStream_t s) {
  return ad.rank <= 16   ? launch_adapter_rp<T, 16, kTaps>(p, map_u, ad, opts, s)
         : ad.rank <= 32 ? launch_adapter_rp<T, 32, kTaps>(p, map_u, ad, opts, s)
                         : launch_adapter_rp<T, 64, kTaps>(p, map_u, ad, opts, s);
}
template <typename T>
cudaError_t launch_adapter_t(const TcPlan& p, const CUtensorMap& map_u, const AdArgs& ad, const LaunchOpts& opts,
                             cudaStream_t s) {
  TcGemmArgs a;
  std::memcpy(&a, p.args, sizeof(a));
  return a.coarse != nullptr && a.cbox_w <= 0 ? launch_adapter_rank<T, true>(p, map_u, ad, opts, s)
                                              : launch_adapter_rank<T, false>(p, map_u, ad, opts, s);
}

int pad8(int v) { return (v + 7) / 8 * 8; }
int store_h(const AdapterProblem& p) { return p.hidden_parts == kAdStored ? kAdFineH : kAdPlain; }
int stored(DType dt, int store) {
  return dt == DType::BF16 ? ad_stored<__nv_bfloat16>(store) : ad_stored<__half>(store);
}
int rank_tile(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Launched ahead of the end of the kernel before on the stream, which the kernel waits for on the device
// before it reads or writes anything (1 to 3 us a call: 143.7 -> 141.6 for P2 of eight images).
LaunchOpts adapter_ahead() {
  LaunchOpts o;
  o.pdl = true;
  return o;
}

// Runs fpn_adapter_split_kernel with S CTAs a tile if they are all resident at once and 4 k-blocks are
// left for each (fewer cost more in the exchange than they save: 2 of rank 64 a CTA on 50 x 76 pixels,
// 16.5 us, 4 of them 14.5 us, as long as unsplit); sets `done`.  Measured, split against not, 16 bits:
// 64 maps of one pixel and K = 2048 14.4 / 22.6 us, 32 of 7 x 7 12.4 / 22.7, two of 50 x 76 with K = 1024
// and a top-down add 14.5 / 16.7; K = 512 12.5 / 12.4.
template <typename T, int RP, int S>
cudaError_t try_adapter_split(const TcPlan& p, const TcGemmArgs& a, const CUtensorMap& map_u, const AdArgs& ad,
                              cudaStream_t s, bool* done) {
  if (a.num_kb < 4 * S || a.num_tiles > sm_count() / S) return cudaSuccess;
  auto kern = fpn_adapter_split_kernel<T, RP, S>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  // (clusters resident at once, the same at every rank: one CTA an SM)
  static std::atomic<int> resident[64];
  int fit = dev < 64 ? resident[dev].load(std::memory_order_acquire) : 0;
  if (fit == 0) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, as_smem(RP).total);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S);
    cfg.blockDim = dim3(kAdThreads);
    cfg.dynamicSmemBytes = as_smem(RP).total;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&fit, kern, &cfg);
    if (e != cudaSuccess) return e;
    if (dev < 64) resident[dev].store(fit, std::memory_order_release);
  }
  if (a.num_tiles > fit) return cudaSuccess;
  *done = true;
  return launch_ex(kern, dim3(a.num_tiles * S), dim3(kAdThreads), as_smem(RP).total, s, adapter_ahead(), S, p.map_a,
                   p.map_b, map_u, a, ad);
}
// The split into the most CTAs a tile that run at once; `done` stays false where none does.
template <typename T, int RP>
cudaError_t launch_adapter_split_rp(const TcPlan& p, const TcGemmArgs& a, const CUtensorMap& map_u, AdArgs ad,
                                    cudaStream_t s, bool* done) {
  ad.h_accs = ad_h_accs((a.num_kb + 7) / 8);
  cudaError_t e = try_adapter_split<T, RP, 8>(p, a, map_u, ad, s, done);
  ad.h_accs = ad_h_accs((a.num_kb + 3) / 4);
  if (e == cudaSuccess && !*done) e = try_adapter_split<T, RP, 4>(p, a, map_u, ad, s, done);
  ad.h_accs = ad_h_accs((a.num_kb + 1) / 2);
  if (e == cudaSuccess && !*done) e = try_adapter_split<T, RP, 2>(p, a, map_u, ad, s, done);
  return e;
}
template <typename T>
cudaError_t launch_adapter_split(const TcPlan& p, const TcGemmArgs& a, const CUtensorMap& map_u, const AdArgs& ad,
                                 cudaStream_t s, bool* done) {
  return ad.rank <= 16   ? launch_adapter_split_rp<T, 16>(p, a, map_u, ad, s, done)
         : ad.rank <= 32 ? launch_adapter_split_rp<T, 32>(p, a, map_u, ad, s, done)
                         : launch_adapter_split_rp<T, 64>(p, a, map_u, ad, s, done);
}

bool adapter_sizes_ok(const AdapterProblem& p) {
  return (p.dtype == DType::BF16 || p.dtype == DType::F16) && p.N > 0 && p.H > 0 && p.W > 0 &&
         p.Cin > 0 && p.Cin % 8 == 0 && p.Cin <= 2048 && p.rank > 0 && p.rank <= kAdMaxRank &&
         p.adapters > 0 && p.adapters <= 65535 &&
         (p.hidden_parts == kAdStored || (p.hidden_parts == 2 && p.dtype == DType::F16)) &&
         static_cast<long long>(p.H) * p.W < ((1LL << 31) - 256) / p.N;
}

// Tiles of a map: with a coarse map the lateral's own 2-D tiles (their taps stay in a small box),
// else runs of 128 pixels of an image taken as one row (fewer padded pixels).
struct AdView {
  int H, W;
  Conv3x3Tiling tiling;
};
AdView adapter_view(const AdapterProblem& p, bool coarse) {
  AdView v;
  if (coarse) {
    v.H = p.H;
    v.W = p.W;
    v.tiling = default_tiling(p.H, p.W);
  } else {
    v.H = 1;
    v.W = p.H * p.W;
    v.tiling.tile_w = 128;
    v.tiling.tile_h = 1;
  }
  return v;
}

// The gradient launch's cut: splits of an image's 64-pixel k-blocks (about one wave of CTAs, at
// least 4 k-blocks each) and images per launch (the partials stay below 256 MB).
struct AgPlan {
  int blocks, x_blocks, num_kb, splits, per, images;
  size_t image_bytes;
};
AgPlan adapter_grad_plan(const AdapterProblem& p) {
  AgPlan g;
  g.x_blocks = (p.Cin + 255) / 256;
  g.blocks = g.x_blocks + 1;
  g.num_kb = static_cast<int>((static_cast<long long>(p.H) * p.W + 63) / 64);
  const long long units = static_cast<long long>(p.N) * g.blocks;
  int k = static_cast<int>(std::max<long long>(1, sm_count() / units));
  k = std::min(k, std::max(1, g.num_kb / 4));
  const int most = (kAdStored * pad8(p.rank) + 15) / 16 * 16 <= 128 ? 32 : 16;  // k-blocks
  g.per = std::min(most, (g.num_kb + k - 1) / k);
  g.splits = (g.num_kb + g.per - 1) / g.per;
  g.image_bytes = static_cast<size_t>(g.splits) * g.blocks * pad8(p.rank) * 256 * sizeof(float);
  g.images = static_cast<int>(std::min<size_t>(p.N, std::max<size_t>(1, (256u << 20) / g.image_bytes)));
  return g;
}

struct AdWorkspace {
  size_t up_t, w_t, dh, part, total;
};
AdWorkspace adapter_workspace(const AdapterProblem& p, bool own_w_t) {
  AdWorkspace w;
  w.up_t = 0;
  w.w_t = w.up_t + align256(static_cast<size_t>(p.adapters) * p.rank * 256 * 2);
  w.dh = w.w_t + (own_w_t ? static_cast<size_t>((p.Cin + 255) / 256) * 256 * 256 * 2 : 0);
  w.part = w.dh + align256(static_cast<size_t>(p.N) * p.H * p.W * kAdStored * pad8(p.rank) * 2);
  const AgPlan g = adapter_grad_plan(p);
  w.total = w.part + g.images * g.image_bytes;
  return w;
}

template <typename T>
cudaError_t adapter_grads_t(const AdapterProblem& p, const void* x, const void* dy, const void* dh,
                            const void* h, float* part, float* ddown, float* dup, int* status,
                            cudaStream_t s) {
  const AgPlan g = adapter_grad_plan(p);
  const int hw = p.H * p.W;
  const int dhc = kAdStored * pad8(p.rank), hc = stored(p.dtype, store_h(p)) * pad8(p.rank);
  CUtensorMap mx, my, mdh, mh;
  cudaError_t e = encode_nhwc_map(&mx, p.dtype, x, p.N, 1, hw, p.Cin, p.Cin, 64, 1);
  if (e == cudaSuccess) e = encode_nhwc_map(&my, p.dtype, dy, p.N, 1, hw, 256, 256, 64, 1);
  if (e == cudaSuccess) e = encode_nhwc_map(&mdh, p.dtype, dh, p.N, 1, hw, dhc, dhc, 64, 1);
  if (e == cudaSuccess) e = encode_nhwc_map(&mh, p.dtype, h, p.N, 1, hw, hc, hc, 64, 1);
  if (e != cudaSuccess) return e;
  auto kern = fpn_adapter_grad_kernel<T>;
  static std::atomic<bool> configured[64];
  e = once_per_device(configured, [&] {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kAgSmemBytes);
  });
  if (e != cudaSuccess) return e;
  const LaunchOpts pdl = adapter_ahead();
  for (int n0 = 0; n0 < p.N; n0 += g.images) {
    const int images = std::min(g.images, p.N - n0);
    AgArgs a;
    std::memset(&a, 0, sizeof(a));
    a.index = p.index;
    a.adapters = p.adapters;
    a.n0 = n0;
    a.splits = g.splits;
    a.per = g.per;
    a.num_kb = g.num_kb;
    a.blocks = g.blocks;
    a.x_blocks = g.x_blocks;
    a.rank_pad = pad8(p.rank);
    a.store = store_h(p);
    a.part = part;
    a.status = status;
    e = launch_ex(kern, dim3(static_cast<unsigned>(images) * g.splits * g.blocks), dim3(kTcThreads),
                  kAgSmemBytes, s, pdl, 1, mx, my, mdh, mh, a);
    if (e != cudaSuccess) return e;
    ArArgs r;
    std::memset(&r, 0, sizeof(r));
    r.index = p.index;
    r.n0 = n0;
    r.images = images;
    r.splits = g.splits;
    r.blocks = g.blocks;
    r.x_blocks = g.x_blocks;
    r.rank = p.rank;
    r.rank_pad = a.rank_pad;
    r.Cin = p.Cin;
    r.part = part;
    r.ddown = ddown;
    r.dup = dup;
    r.more = n0 > 0;
    e = launch_ex(adapter_reduce_kernel, dim3(g.blocks * p.rank, p.adapters), dim3(256), 0, s, pdl, 1, r);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// 16-bit parts of the bilinear weights on the tensor cores: one where they are exact (ratios of 1 to 8 that are
// powers of two: products of the axes' 0, 2, 3 or 4 bits), else two, 16 bits and more of a weight.  (One rounded
// part left a constant coarse map up to 2.9e-3 off in bf16; two cost 6 % on two 200 x 304 maps over 67 x 102.)
int bilinear_parts(int H, int W, int Hc, int Wc) {
  auto bits = [](int out, int in) {
    return out == in ? 0 : out == 2 * in ? 2 : out == 4 * in ? 3 : out == 8 * in ? 4 : 16;
  };
  return bits(H, Hc) + bits(W, Wc) <= 8 ? 1 : 2;
}

}  // namespace

cudaError_t launch_lateral_adapters(const AdapterProblem& p, const void* x, const void* w,
                                    const float* bias, const void* down, const void* up,
                                    const void* coarse, int Hc, int Wc, void* out, void* hidden,
                                    int* status, cudaStream_t s) {
  if (!adapter_sizes_ok(p)) return cudaErrorInvalidValue;
  CUtensorMap map_u;
  cudaError_t e =
      encode_nhwc_map(&map_u, p.dtype, down, p.adapters, 1, p.rank, p.Cin, p.Cin, rank_tile(p.rank), 1);
  if (e != cudaSuccess) return e;
  AdArgs ad;
  std::memset(&ad, 0, sizeof(ad));
  ad.index = p.index;
  ad.scales = p.scales;
  ad.scale = p.scale;
  ad.adapters = p.adapters;
  ad.rank = p.rank;
  ad.v = up;
  ad.va = 256LL * p.rank;
  ad.vc = p.rank;
  ad.vr = 1;
  ad.v_rows = 256;
  ad.v_vec = p.rank % 8 == 0 && aligned16(up);
  ad.hidden = hidden;
  ad.store = store_h(p);
  ad.rank_pad = pad8(p.rank);
  ad.want_out = 1;
  ad.h_accs = ad_h_accs((p.Cin + 63) / 64);
  ad.out = out;
  ad.out_c = 256;
  ad.map_h = p.H;
  ad.map_w = p.W;
  ad.bil_parts = coarse ? bilinear_parts(p.H, p.W, Hc, Wc) : 1;
  TcPlan plan;
  // Few tiles: split over k (at most half the SMs, so that two CTAs a tile fit).
  if ((p.Cin + 63) / 64 >= 8 &&
      (static_cast<long long>(p.H) * p.W + kTcBlockM - 1) / kTcBlockM * p.N <= sm_count() / 2) {
    const AdView v = adapter_view(p, false);
    e = plan_tc_lateral(plan, p.dtype, x, w, bias, nullptr, out, p.N, p.Cin, v.H, v.W, 0, 0, v.tiling, status, 0);
    if (e != cudaSuccess) return e;
    TcGemmArgs a;
    std::memcpy(&a, plan.args, sizeof(a));
    if (coarse) {
      a.coarse = coarse;
      a.Hc = Hc;
      a.Wc = Wc;
      a.scale_y = static_cast<float>(Hc) / static_cast<float>(p.H);
      a.scale_x = static_cast<float>(Wc) / static_cast<float>(p.W);
    }
    bool done = false;
    e = p.dtype == DType::BF16 ? launch_adapter_split<__nv_bfloat16>(plan, a, map_u, ad, s, &done)
                               : launch_adapter_split<__half>(plan, a, map_u, ad, s, &done);
    if (e != cudaSuccess || done) return e;
  }
  const AdView v = adapter_view(p, coarse != nullptr);
  e = plan_tc_lateral(plan, p.dtype, x, w, bias, coarse, out, p.N, p.Cin, v.H, v.W, Hc, Wc, v.tiling, status, 0);
  if (e != cudaSuccess) return e;
  return p.dtype == DType::BF16 ? launch_adapter_t<__nv_bfloat16>(plan, map_u, ad, adapter_ahead(), s)
                                : launch_adapter_t<__half>(plan, map_u, ad, adapter_ahead(), s);
}

size_t lateral_adapters_workspace_bytes(const AdapterProblem& p, bool has_w_t, bool need_dx) {
  return adapter_sizes_ok(p) ? adapter_workspace(p, need_dx && !has_w_t).total : 0;
}

cudaError_t launch_lateral_adapters_backward(const AdapterProblem& p, const void* x, const void* w,
                                             const void* w_t, const void* dy, const void* down,
                                             const void* up, const void* hidden, void* dx, float* ddown,
                                             float* dup, void* ws, size_t ws_bytes, int* status,
                                             cudaStream_t s) {
  if (!adapter_sizes_ok(p)) return cudaErrorInvalidValue;
  const AdWorkspace wl = adapter_workspace(p, dx != nullptr && !w_t);
  if (ws_bytes < wl.total) return cudaErrorInvalidValue;
  uint8_t* base = static_cast<uint8_t*>(ws);
  void* up_t = base + wl.up_t;
  void* dh = base + wl.dh;
  const int slices = (p.Cin + 255) / 256;
  const bool own_w_t = dx && !w_t;
  cudaError_t e = launch_ex(adapter_transpose_kernel, dim3(p.adapters + (own_w_t ? slices * 8 : 0)), dim3(256), 0, s,
                            LaunchOpts(), 1, static_cast<const uint16_t*>(up), static_cast<uint16_t*>(up_t), p.rank,
                            p.adapters, static_cast<const uint16_t*>(w), reinterpret_cast<uint16_t*>(base + wl.w_t),
                            p.Cin);
  if (e != cudaSuccess) return e;
  if (own_w_t) w_t = base + wl.w_t;
  const AdView v = adapter_view(p, false);
  TcPlan plan;
  // (without dx the output and weight maps are unused: any valid tensors)
  e = plan_tc_lateral(plan, p.dtype, dy, dx ? w_t : up_t, nullptr, nullptr, dx ? dx : dh, p.N, 256, v.H,
                      v.W, 0, 0, v.tiling, status, 0);
  if (e == cudaSuccess && dx) e = tc_set_channel_slices(plan, w_t, 256, slices, dx, p.Cin);
  if (e != cudaSuccess) return e;
  CUtensorMap map_u;
  e = encode_nhwc_map(&map_u, p.dtype, up_t, p.adapters, 1, p.rank, 256, 256, rank_tile(p.rank), 1);
  if (e != cudaSuccess) return e;
  AdArgs ad;
  std::memset(&ad, 0, sizeof(ad));
  ad.index = p.index;
  ad.scales = p.scales;
  ad.scale = p.scale;
  ad.adapters = p.adapters;
  ad.rank = p.rank;
  ad.v = down;
  ad.va = static_cast<long long>(p.rank) * p.Cin;
  ad.vc = 1;
  ad.vr = p.Cin;
  ad.v_rows = p.Cin;
  ad.hidden = dh;
  ad.store = kAdFineDh;
  ad.rank_pad = pad8(p.rank);
  ad.want_out = dx != nullptr;
  ad.h_accs = ad_h_accs(4);
  ad.bil_parts = 1;
  ad.out = dx;
  ad.out_c = p.Cin;
  e = p.dtype == DType::BF16 ? launch_adapter_t<__nv_bfloat16>(plan, map_u, ad, adapter_ahead(), s)
                             : launch_adapter_t<__half>(plan, map_u, ad, adapter_ahead(), s);
  if (e != cudaSuccess) return e;
  float* part = reinterpret_cast<float*>(base + wl.part);
  return p.dtype == DType::BF16
             ? adapter_grads_t<__nv_bfloat16>(p, x, dy, dh, hidden, part, ddown, dup, status, s)
             : adapter_grads_t<__half>(p, x, dy, dh, hidden, part, ddown, dup, status, s);
}

}  // namespace ufpn
