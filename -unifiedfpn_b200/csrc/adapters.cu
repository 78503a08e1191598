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
// h is kept in two 16-bit parts, hi = round(h) and lo = round(h - hi), 16 (bf16) or 22 (fp16) bits
// together: one rounding to bf16 would be the largest error of the fp32 weight gradients, and of
// an adapter's share of out, for one k-step more.  The backward reads both parts.
#include "kernels.h"
#include "tc_gemm.cuh"

#include <algorithm>
#include <atomic>
#include <cstring>

namespace ufpn {

namespace {

constexpr int kAdMaxRank = 64;
constexpr int kAdThreads = kTcThreads;  // TMA warp, MMA warp, 8 epilogue warps
constexpr int kDevTimeoutAdapter = 0x107;

// Shared memory of fpn_adapter_kernel for ranks up to RP.
template <int RP>
struct AdCfg {
  static constexpr int kU = RP * 128;  // one k-block of down[a]
  static constexpr int kStage = kTcAStage + kTcBStage + kU;
  static constexpr int kStages = RP <= 32 ? 3 : 2;  // (three of 56 KB would not fit)
  static constexpr int kOffV = kStages * kStage;         // up[a]: 256 rows of 128 bytes
  static constexpr int kOffT = kOffV + kTcBStage;        // h: hi, lo; then the output's staging
  static constexpr int kOffBars = kOffT + 2 * kTcAStage;
  static constexpr int kSmemBytes = kOffBars + 256 + 1024 /*alignment slack*/;
  static_assert(kU % 1024 == 0 && kSmemBytes <= 232448, "adapter smem");
  static_assert(2 * kTcAStage == kTcEpiWarps * kTcStagingPerWarp, "staging takes h's place");
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
  void* hidden;  // [pixels][2][rank_pad] hi, lo; or null
  int rank_pad;  // rank rounded up to 8
  int want_out;  // 0: only hidden
};

__device__ __forceinline__ int ad_adapter(const AdArgs& a, int n) {
  const int i = __ldg(a.index + n);
  return i >= 0 && i < a.adapters ? i : -1;
}

// h in two parts: v ~ hi + lo.  (fp16: a value beyond its range keeps the rest in lo.)
template <typename T>
__device__ __forceinline__ void ad_split(float v, uint16_t& hi, uint16_t& lo) {
  float c = v;
  if constexpr (TcElem<T>::kFmt == 0) c = v > 65504.f ? 65504.f : (v < -65504.f ? -65504.f : v);
  hi = Pack<T>::bits(c);
  const float h = Pack<T>::unpack(static_cast<uint32_t>(hi)).x;
  lo = Pack<T>::bits(v - h);
}

template <typename T, int RP>
__global__ void __launch_bounds__(kAdThreads, 1)
    fpn_adapter_kernel(const __grid_constant__ CUtensorMap map_a,
                       const __grid_constant__ CUtensorMap map_b,
                       const __grid_constant__ CUtensorMap map_out,
                       const __grid_constant__ CUtensorMap map_coarse,
                       const __grid_constant__ CUtensorMap map_u, const TcGemmArgs args,
                       const AdArgs ad) {
  using Cfg = AdCfg<RP>;
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
  uint64_t* sfree_bar = accf_bar + 4;  // every warp's stores have left the staging
  uint64_t* done_bar = accf_bar + 5;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const bool bil_mma = args.coarse != nullptr && args.cbox_w > 0;
  constexpr uint32_t kHCol = kTcBlockN;  // h accumulator: TMEM columns [256, 256 + RP)

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(accf_bar, 1);
    mbar_init(acce_bar, kTcEpiWarps * 32);
    mbar_init(hfull_bar, 1);
    mbar_init(tfull_bar, kTcEpiWarps * 32);
    mbar_init(sfree_bar, kTcEpiWarps);
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
    prefetch_tmap(&map_u);
    prefetch_tmap(&map_out);
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
    const uint32_t coarse_bytes = static_cast<uint32_t>(args.cbox_w * args.cbox_h * 128 * 4);
    for (int tile = blockIdx.x; ok && tile < args.num_tiles; tile += gridDim.x) {
      int n, x0, y0, slice;
      tc_tile_origin(args, tile, n, x0, y0, slice);
      const int adapter = ad_adapter(ad, n);
      if (!ad.want_out && adapter < 0) continue;
      const int nkb = args.num_kb + (bil_mma ? 1 : 0);
      for (int kb = 0; kb < nkb; ++kb) {
        ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, args.status, kDevTimeoutAdapter);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        uint8_t* const sa = smem + stage * Cfg::kStage;
        uint8_t* const sb = sa + kTcAStage;
        uint8_t* const su = sb + kTcBStage;
        if (kb < args.num_kb) {
          if (lane == 0) {
            mbar_arrive_expect_tx(&full_bar[stage], kTcAStage + (ad.want_out ? kTcBStage : 0) +
                                                        (adapter >= 0 ? Cfg::kU : 0));
            tma_load_4d(sa, &map_a, &full_bar[stage], kb * 64, x0, y0, n, kPolicyEvictFirst);
            if (ad.want_out)
              tma_load_2d(sb, &map_b, &full_bar[stage], kb * 64, slice * kTcBlockN, kPolicyEvictLast);
            if (adapter >= 0)
              tma_load_4d(su, &map_u, &full_bar[stage], kb * 64, 0, 0, adapter, kPolicyEvictLast);
          }
        } else {
          // top-down k-block, as in the plain lateral
          tc_build_bilinear<T>(sa, sb, lane, x0, y0, args.tile_w, args.H, args.W, args.Hc, args.Wc,
                               args.scale_y, args.scale_x, args.cbox_w, args.cbox_h);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            const int cy = static_cast<int>(tc_src(y0, args.scale_y, args.Hc));
            const int cx = static_cast<int>(tc_src(x0, args.scale_x, args.Wc));
            mbar_arrive_expect_tx(&full_bar[stage], coarse_bytes);
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
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < args.num_tiles; tile += gridDim.x) {
        int n, x0, y0, slice;
        tc_tile_origin(args, tile, n, x0, y0, slice);
        const bool has = ad_adapter(ad, n) >= 0;
        if (!ad.want_out && !has) continue;
        if (!mbar_wait(acce_bar, tile_phase ^ 1u, abort_flag, args.status, kDevTimeoutAdapter)) break;
        tc_fence_after();
        const int nkb = args.num_kb + (bil_mma ? 1 : 0);
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
            const uint64_t udesc = sdesc_kmajor_sw128(sa + kTcAStage + kTcBStage);
#pragma unroll
            for (int k = 0; k < kMmaPerKb; ++k) {
              const uint32_t acc = (kb > 0 || k > 0) ? 1u : 0u;
              if (ad.want_out) tc_mma_f16(tmem_base, adesc + 2u * k, bdesc + 2u * k, idesc, acc);
              if (has) tc_mma_f16(tmem_base + kHCol, adesc + 2u * k, udesc + 2u * k, idesc_u, acc);
            }
          } else {
            const uint64_t bdesc = sdesc_mnmajor_sw128(sa + kTcAStage, kTcCoarseMaxPix * 128);
#pragma unroll
            for (int k = 0; k < kMmaPerKb; ++k)
              tc_mma_f16(tmem_base, adesc + 2u * k, bdesc + 128u * k, idesc_bmn, 1u);
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
            if (!mbar_wait(tfull_bar, h_phase, abort_flag, args.status, kDevTimeoutAdapter)) break;
            tc_fence_after();
            const uint32_t t = smem_u32(smem + Cfg::kOffT);
            const uint64_t vdesc = sdesc_kmajor_sw128(smem_u32(smem + Cfg::kOffV));
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              const uint64_t tdesc = sdesc_kmajor_sw128(t + part * kTcAStage);
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
      tc_commit(done_bar);
      mbar_wait_drain(done_bar, 0);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - 2;
    const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31
    const int chalf = ew >> 2;     // output channels 128 * chalf .. + 127
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    uint8_t* const my_stage = smem + Cfg::kOffT + ew * kTcStagingPerWarp;
    const int tw = args.tile_w;
    const bool taps_global = args.coarse != nullptr && !bil_mma;
    uint32_t tile_phase = 0, h_phase = 0;
    int v_adapter = -1, v_slice = -1;  // what the up region holds
    for (int tile = blockIdx.x; tile < args.num_tiles; tile += gridDim.x) {
      int n, x0, y0, slice;
      tc_tile_origin(args, tile, n, x0, y0, slice);
      const int adapter = ad_adapter(ad, n);
      const bool has = adapter >= 0;
      const int py = y0 + row / tw, px = x0 + row % tw;
      const bool valid = py < args.H && px < args.W;
      uint4* hid = nullptr;  // this thread's pixel of `hidden`: 2 * rank_pad elements
      if (ad.hidden != nullptr && slice == 0 && valid && chalf == 0)
        hid = reinterpret_cast<uint4*>(
            static_cast<uint8_t*>(ad.hidden) +
            ((static_cast<size_t>(n) * args.H + py) * args.W + px) * ad.rank_pad * 4);
      if (has) {
        if (lane == 0) {
          bulk_wait_group_read<0>();
          mbar_arrive(sfree_bar);
        }
        __syncwarp();
        if (chalf == 1 && ad.want_out && (adapter != v_adapter || slice != v_slice)) {
          // up[a] (this slice's 256 rows): the MMA that read the last one has completed (this
          // thread has waited for its accumulator)
          const uint16_t* v = static_cast<const uint16_t*>(ad.v) + adapter * ad.va;
          const uint32_t dst = smem_u32(smem + Cfg::kOffV);
          const int e = (ew - 4) * 32 + lane;
#pragma unroll 1
          for (int c = e; c < kTcBlockN; c += 128) {
            const int ch = slice * kTcBlockN + c;
            const uint16_t* src = v + ch * ad.vc;
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
              st_shared_v4(dst + c * 128 + ((j ^ (c & 7)) << 4), q);
            }
          }
        }
        if (chalf == 1) {
          v_adapter = adapter;
          v_slice = slice;
        }
        // (every warp waits for the tile's h, so that none runs ahead on the barriers below)
        bool ok = mbar_wait(hfull_bar, h_phase, abort_flag, args.status, kDevTimeoutAdapter);
        if (chalf == 0)
          ok = ok && mbar_wait(sfree_bar, h_phase, abort_flag, args.status, kDevTimeoutAdapter);
        ok = __all_sync(0xffffffffu, ok);
        if (chalf == 0) {
          if (ok) {
            tc_fence_after();
            const float s = ad.scale * (ad.scales != nullptr ? __ldg(ad.scales + adapter) : 1.f);
            const uint32_t t = smem_u32(smem + Cfg::kOffT) + row * 128;
#pragma unroll
            for (int j = 0; j < RP / 8; ++j) {
              uint32_t r[8];
              __syncwarp();
              tmem_ld8(tmem_base + kHCol + j * 8 + lane_addr, r);
              tmem_wait_ld();
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint16_t h0, l0, h1, l1;
                const int c = j * 8 + 2 * i;
                ad_split<T>(c < ad.rank ? s * __uint_as_float(r[2 * i]) : 0.f, h0, l0);
                ad_split<T>(c + 1 < ad.rank ? s * __uint_as_float(r[2 * i + 1]) : 0.f, h1, l1);
                hi[i] = h0 | (static_cast<uint32_t>(h1) << 16);
                lo[i] = l0 | (static_cast<uint32_t>(l1) << 16);
              }
              const uint4 qh = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              const uint4 ql = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              const uint32_t off = static_cast<uint32_t>((j ^ (row & 7)) << 4);
              if (ad.want_out) {
                st_shared_v4(t + off, qh);
                st_shared_v4(t + kTcAStage + off, ql);
              }
              if (hid != nullptr && j * 8 < ad.rank_pad) {
                hid[j] = qh;
                hid[ad.rank_pad / 8 + j] = ql;
              }
            }
          }
        }
        if (!ok) break;
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(tfull_bar);
        h_phase ^= 1u;
        if (!ad.want_out) mbar_arrive(acce_bar);
      } else if (hid != nullptr) {
        for (int j = 0; j < ad.rank_pad / 4; ++j) hid[j] = make_uint4(0u, 0u, 0u, 0u);
      }
      if (!ad.want_out) continue;

      const bool ok = mbar_wait(accf_bar, tile_phase, abort_flag, args.status, kDevTimeoutAdapter);
      if (!__all_sync(0xffffffffu, ok)) break;
      tile_phase ^= 1u;
      tc_fence_after();
      // The whole accumulator row goes to registers at once, so that the next tile's MMAs start
      // while this one is converted and stored.
      uint32_t rr[128];
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 4; ++q)
        tmem_ld32(tmem_base + chalf * 128 + q * 32 + lane_addr,
                  *reinterpret_cast<uint32_t(*)[32]>(&rr[q * 32]));
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(acce_bar);

      TcTaps tp{};
      const uint8_t* cb = nullptr;
      size_t o00 = 0, o01 = 0, o10 = 0, o11 = 0;
      if (taps_global) {
        tp = tc_taps(py, px, args.H, args.W, args.Hc, args.Wc, args.scale_y, args.scale_x);
        constexpr size_t rowb = kTcBlockN * 2;
        cb = static_cast<const uint8_t*>(args.coarse) + static_cast<size_t>(n) * args.Hc * args.Wc * rowb;
        o00 = (static_cast<size_t>(tp.ya) * args.Wc + tp.xa) * rowb;
        o01 = (static_cast<size_t>(tp.ya) * args.Wc + tp.xb) * rowb;
        o10 = (static_cast<size_t>(tp.yb) * args.Wc + tp.xa) * rowb;
        o11 = (static_cast<size_t>(tp.yb) * args.Wc + tp.xb) * rowb;
      }
      const int ox = x0 + (quarter * 32) % tw, oy = y0 + (quarter * 32) / tw;
      const int scol = slice * kTcBlockN;
      const uint32_t stage_addr = smem_u32(my_stage) + lane * 128;
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        const int col0 = chalf * 128 + step * 64;
        if (lane == 0) bulk_wait_group_read<0>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float v[8];
          const int c = col0 + j * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(rr[step * 64 + j * 8 + i]);
          if (args.bias != nullptr) {
            const float4 b0 = __ldg(reinterpret_cast<const float4*>(args.bias + scol + c));
            const float4 b1 = __ldg(reinterpret_cast<const float4*>(args.bias + scol + c) + 1);
            v[0] += b0.x, v[1] += b0.y, v[2] += b0.z, v[3] += b0.w;
            v[4] += b1.x, v[5] += b1.y, v[6] += b1.z, v[7] += b1.w;
          }
          if (taps_global) {
            const uint4 q[4] = {__ldg(reinterpret_cast<const uint4*>(cb + o00 + c * 2)),
                                __ldg(reinterpret_cast<const uint4*>(cb + o01 + c * 2)),
                                __ldg(reinterpret_cast<const uint4*>(cb + o10 + c * 2)),
                                __ldg(reinterpret_cast<const uint4*>(cb + o11 + c * 2))};
            const float w[4] = {tp.w00, tp.w01, tp.w10, tp.w11};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t u[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = Pack<T>::unpack(u[e]);
                v[2 * e] = fmaf(w[k], f.x, v[2 * e]);
                v[2 * e + 1] = fmaf(w[k], f.y, v[2 * e + 1]);
              }
            }
          }
          st_shared_v4(stage_addr + ((j ^ (lane & 7)) << 4),
                       make_uint4(Pack<T>::pack(v[0], v[1]), Pack<T>::pack(v[2], v[3]),
                                  Pack<T>::pack(v[4], v[5]), Pack<T>::pack(v[6], v[7])));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (args.out_cols == 0 || scol + col0 < args.out_cols)
            tma_store_4d(&map_out, my_stage, scol + col0, ox, oy, n);
          bulk_commit_group();
        }
      }
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, kTcTmemCols);
  }
}

// ------------------------------------------------------------------ adapter gradients
// part[unit][r][c] = sum over the unit's pixels of h[p][r] q[p][c], h = hi + lo: for the channel
// blocks of x with h = dh (ddown), and for dy with h (dup).  A tcgen05 GEMM over pixels (both
// operands MN-major 64-pixel boxes): M = 256 channels in two accumulators, N = 2 rank_pad columns,
// the hi and lo parts side by side, added when the accumulators are read.
constexpr int kAgChunk = 64 * 128;
constexpr int kAgStages = 4;
constexpr int kAgQ = 4 * kAgChunk;                 // 256 channels
constexpr int kAgStage = kAgQ + 2 * kAgChunk;      // + up to 128 columns of h
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
  float* part;  // [image - n0][split][block][rank_pad][256]
  int* status;
};

template <typename T>
__global__ void __launch_bounds__(kAdThreads, 1)
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
  if (adapter < 0 || adapter >= a.adapters) return;  // (before any barrier or TMEM)

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
  const int cols = 2 * a.rank_pad;
  const int hchunks = (cols + 63) / 64;

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
    tmem_alloc(tmem_slot, 256);
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
          const uint32_t acc = (kb > kb0 || k > 0) ? 1u : 0u;
          tc_mma_f16(tmem_base, a0 + 128u * k, b + 128u * k, idesc, acc);
          tc_mma_f16(tmem_base + 128, a1 + 128u * k, b + 128u * k, idesc, acc);
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
      const uint32_t acc = tmem_base + half * 128 + (static_cast<uint32_t>(quarter * 32) << 16);
      float* dst = a.part + ((static_cast<size_t>(n - a.n0) * a.splits + split) * a.blocks + block) *
                                a.rank_pad * 256 +
                   half * 128 + quarter * 32 + lane;
      for (int r = 0; r < a.rank_pad; r += 8) {
        uint32_t hi[8], lo[8];
        __syncwarp();
        tmem_ld8(acc + r, hi);
        tmem_ld8(acc + a.rank_pad + r, lo);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          dst[(r + i) * 256] = __uint_as_float(hi[i]) + __uint_as_float(lo[i]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
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

// up [L][256][R] -> [L][R][256]
__global__ void __launch_bounds__(256) adapter_transpose_kernel(const uint16_t* __restrict__ up,
                                                                uint16_t* __restrict__ out, int rank) {
  const size_t a = blockIdx.x;
  for (int r = 0; r < rank; ++r)
    out[(a * rank + r) * 256 + threadIdx.x] = up[(a * 256 + threadIdx.x) * rank + r];
}

// ------------------------------------------------------------------ host side
template <typename T, int RP>
cudaError_t launch_adapter_rp(const TcPlan& p, const CUtensorMap& map_u, const AdArgs& ad, cudaStream_t s) {
  using Cfg = AdCfg<RP>;
  auto kern = fpn_adapter_kernel<T, RP>;
  static std::atomic<bool> configured[64];
  cudaError_t e = once_per_device(configured, [&] {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
  });
  if (e != cudaSuccess) return e;
  TcGemmArgs a;
  std::memcpy(&a, p.args, sizeof(a));
  return launch_ex(kern, dim3(p.grid), dim3(kAdThreads), Cfg::kSmemBytes, s, LaunchOpts(), 1, p.map_a,
                   p.map_b, p.map_out, p.map_coarse, map_u, a, ad);
}
template <typename T>
cudaError_t launch_adapter_t(const TcPlan& p, const CUtensorMap& map_u, const AdArgs& ad, cudaStream_t s) {
  if (ad.rank <= 16) return launch_adapter_rp<T, 16>(p, map_u, ad, s);
  if (ad.rank <= 32) return launch_adapter_rp<T, 32>(p, map_u, ad, s);
  return launch_adapter_rp<T, 64>(p, map_u, ad, s);
}

int pad8(int v) { return (v + 7) / 8 * 8; }
int rank_tile(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

bool adapter_sizes_ok(const AdapterProblem& p) {
  return (p.dtype == DType::BF16 || p.dtype == DType::F16) && p.N > 0 && p.H > 0 && p.W > 0 &&
         p.Cin > 0 && p.Cin % 8 == 0 && p.Cin <= 2048 && p.rank > 0 && p.rank <= kAdMaxRank &&
         p.adapters > 0 && p.adapters <= 65535 && static_cast<long long>(p.H) * p.W < (1LL << 31) - 256;
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
  g.per = (g.num_kb + k - 1) / k;
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
  w.part = w.dh + align256(static_cast<size_t>(p.N) * p.H * p.W * 2 * pad8(p.rank) * 2);
  const AgPlan g = adapter_grad_plan(p);
  w.total = w.part + g.images * g.image_bytes;
  return w;
}

template <typename T>
cudaError_t adapter_grads_t(const AdapterProblem& p, const void* x, const void* dy, const void* dh,
                            const void* h, float* part, float* ddown, float* dup, int* status,
                            cudaStream_t s) {
  const AgPlan g = adapter_grad_plan(p);
  const int hw = p.H * p.W, hc = 2 * pad8(p.rank);
  CUtensorMap mx, my, mdh, mh;
  cudaError_t e = encode_nhwc_map(&mx, p.dtype, x, p.N, 1, hw, p.Cin, p.Cin, 64, 1);
  if (e == cudaSuccess) e = encode_nhwc_map(&my, p.dtype, dy, p.N, 1, hw, 256, 256, 64, 1);
  if (e == cudaSuccess) e = encode_nhwc_map(&mdh, p.dtype, dh, p.N, 1, hw, hc, hc, 64, 1);
  if (e == cudaSuccess) e = encode_nhwc_map(&mh, p.dtype, h, p.N, 1, hw, hc, hc, 64, 1);
  if (e != cudaSuccess) return e;
  auto kern = fpn_adapter_grad_kernel<T>;
  static std::atomic<bool> configured[64];
  e = once_per_device(configured, [&] {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kAgSmemBytes);
  });
  if (e != cudaSuccess) return e;
  LaunchOpts pdl;
  pdl.pdl = true;
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
    a.part = part;
    a.status = status;
    e = launch_ex(kern, dim3(static_cast<unsigned>(images) * g.splits * g.blocks), dim3(kAdThreads),
                  kAgSmemBytes, s, LaunchOpts(), 1, mx, my, mdh, mh, a);
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
    e = launch_ex(adapter_reduce_kernel, dim3(g.blocks * p.rank, p.adapters), dim3(256), 0, s,
                  LaunchOpts(), 1, r);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_lateral_adapters(const AdapterProblem& p, const void* x, const void* w,
                                    const float* bias, const void* down, const void* up,
                                    const void* coarse, int Hc, int Wc, void* out, void* hidden,
                                    int* status, cudaStream_t s) {
  if (!adapter_sizes_ok(p)) return cudaErrorInvalidValue;
  const AdView v = adapter_view(p, coarse != nullptr);
  TcPlan plan;
  cudaError_t e = plan_tc_lateral(plan, p.dtype, x, w, bias, coarse, out, p.N, p.Cin, v.H, v.W, Hc, Wc,
                                  v.tiling, status, 0);
  if (e != cudaSuccess) return e;
  CUtensorMap map_u;
  e = encode_nhwc_map(&map_u, p.dtype, down, p.adapters, 1, p.rank, p.Cin, p.Cin, rank_tile(p.rank), 1);
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
  ad.rank_pad = pad8(p.rank);
  ad.want_out = 1;
  return p.dtype == DType::BF16 ? launch_adapter_t<__nv_bfloat16>(plan, map_u, ad, s)
                                : launch_adapter_t<__half>(plan, map_u, ad, s);
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
  cudaError_t e = launch_ex(adapter_transpose_kernel, dim3(p.adapters), dim3(256), 0, s, LaunchOpts(), 1,
                            static_cast<const uint16_t*>(up), static_cast<uint16_t*>(up_t), p.rank);
  if (e != cudaSuccess) return e;
  const int slices = (p.Cin + 255) / 256;
  if (dx && !w_t) {
    if ((e = launch_transpose_weights(p.dtype, w, base + wl.w_t, 256, p.Cin, slices * 256, s)) != cudaSuccess)
      return e;
    w_t = base + wl.w_t;
  }
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
  ad.rank_pad = pad8(p.rank);
  ad.want_out = dx != nullptr;
  e = p.dtype == DType::BF16 ? launch_adapter_t<__nv_bfloat16>(plan, map_u, ad, s)
                             : launch_adapter_t<__half>(plan, map_u, ad, s);
  if (e != cudaSuccess) return e;
  float* part = reinterpret_cast<float*>(base + wl.part);
  return p.dtype == DType::BF16
             ? adapter_grads_t<__nv_bfloat16>(p, x, dy, dh, hidden, part, ddown, dup, status, s)
             : adapter_grads_t<__half>(p, x, dy, dh, hidden, part, ddown, dup, status, s);
}

}  // namespace ufpn
