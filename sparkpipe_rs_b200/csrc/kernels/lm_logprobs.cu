// Log probabilities of given tokens and entropy straight from hidden states x [T, K] and the
// LM head's weight w [V, K] (bf16): logits = x w^T exist only as tcgen05 accumulators, sm_100a.
//
// For a row of logits l: m = max l, S = sum exp(l_i - m), E = sum exp(l_i - m) (l_i - m);
//   log p_i = (l_i - m) - ln S,   entropy = ln S - E / S.
// A CTA walks the vocabulary tiles of its share for 128 rows, tile by tile 128 x 256 logits in
// tensor memory, and its epilogue threads (one row of half a tile each) keep m, S, E and the
// given token's logit running; a second kernel joins the shares of a row. The logits of an
// 8,192-token chunk over 102,400 tokens would be 3.4 GB in fp32.
//
// What bounds it: the products for many rows (2 T V K operations), one read of w for few.
//
//  * The tensor cores add the products of a K block onto the accumulator and cut the sum off
//    below its last bit instead of rounding: over long K the logits shrink by about 1e-6 of
//    their size, all the same way, which shows in the entropy (off by 1.5e-6 of itself at K =
//    2,048). So K is taken in segments, each with an accumulator of its own, and the epilogue
//    adds the segments with rounding. Off from 64 bits (2-norm, logits of variance 6): segments
//    of 512 3e-7 to 4.5e-7, of 256, where one row tile leaves the epilogue idle anyway, 1.2e-7 to
//    1.7e-7 (a single row up to 2.4e-7), of 1,024 6e-7 to 1e-6, the less the more tokens there
//    are. On CTA pairs each pass of the epilogue costs: segments of 1,024 are 5 to 9% faster than
//    of 512 whatever the number of rows and tokens (150 x 32,768 x 2,048 34.8 us, 38.1; 8,192 x
//    102,400 x 2,048 at the power limit 2.45 ms, 2.60; K = 7,168 0 to 4%). They are taken from 32,768 tokens on, where
//    they keep the entropy within 9e-7 (10,000 tokens: 1e-6).
//  * Work items are (128 rows, a range of 64-token units of the vocabulary), rows fastest:
//    the CTAs that run at the same time read the same range of w, so it comes from memory
//    once and then from L2, and one row tile's shares are few enough to join cheaply.
//  * Warp roles (320 threads): warp 0 TMA, warp 1 MMA and tensor memory, warps 2..9 epilogue
//    (lane quarter = warp % 4, columns [0, 128) or [128, 256) of a tile).
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "common.cuh"
#include "launch.h"
#include "logprobs.cuh"
#include "pdl.h"

namespace sp {

namespace {

constexpr int kRows = kLmRows;
constexpr int kCols = 256;       // logits of a tile's row
constexpr int kBox = 64;         // rows of a TMA box of w
constexpr int kBlockK = 64;
constexpr int kXBytes = kRows * kBlockK * 2;
constexpr int kBoxBytes = kBox * kBlockK * 2;
constexpr int kHalf = 128;       // columns of an epilogue thread
constexpr int kEpilogue = 256;   // epilogue threads
constexpr int kManyTokens = 32768;  // pairs take long segments of K from here on

// CTAs = 2: a pair of CTAs shares a tile of 256 rows x 256 logits, each loads half of w's rows.
template <int CTAS>
struct Lm {
  static constexpr int kUnit = kBox * CTAS;         // tokens of a unit of the vocabulary
  static constexpr int kTile = kCols / kUnit;       // units of a tile = boxes of w that a CTA loads
};

// The ring holds as many stages as fit: a stage is the rows of x that there are and the boxes of
// the largest tile, 48 KB for 128 x 256, 10 KB for a few rows and a share of 64 tokens.
constexpr int kMaxStages = 16;
constexpr int kRing = 224 * 1024;
constexpr int kSmem = kRing + 1024 + 512;
static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");

struct LmParams {
  int T, V, K;
  int row_tiles, units, shares;  // row tiles, units of the vocabulary, shares of a row tile
  int x_bytes;                   // of a box of x: one row tile loads only the rows that there are
  int block_bytes;               // of a K block in the ring: x and the boxes of w
  int stages, stage_bytes;
  const int* ids;
  float4* part;                  // [shares * 2][row_tiles * 128]: m, S, E (log2 units), the given token's logit
  int* err;
};

SP_DEVI void share_units(const LmParams& p, int share, int& u0, int& u1) {
  u0 = int((long long)p.units * share / p.shares);
  u1 = int((long long)p.units * (share + 1) / p.shares);
}

// Units of the next tile: a share's tiles are alike (five units go as 3 + 2: a K block of one unit
// takes a CTA as long as one of two).
template <int TILE>
SP_DEVI int next_tile(int left) {
  const int tiles = (left + TILE - 1) / TILE;
  return (left + tiles - 1) / tiles;
}

}  // namespace

// SEG: K blocks of a segment, PER: of a stage of the ring.
template <int CTAS, int SEG, int PER>
__global__ void __launch_bounds__(64 + kEpilogue, 1)
    lm_logprobs_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                       const LmParams p) {
  using C = Lm<CTAS>;
  constexpr int kTile = C::kTile, kUnit = C::kUnit;
  const int stages = p.stages, stage_bytes = p.stage_bytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kRing);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* s_err = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 2 ? (int)cluster_ctarank() : 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], CTAS * kEpilogue / 32);
    }
    *s_err = 0;
    fence_mbarrier_init();
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmW);
  }
  if (warp == 1) {
    if (CTAS == 2) {
      tmem_alloc_pair<2 * kCols>(tmem_slot);
      tmem_relinquish_pair();
    } else {
      tmem_alloc<2 * kCols>(tmem_slot);
      tmem_relinquish();
    }
    tc_fence_before();
  }
  if (CTAS == 2) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  griddep_launch();
  griddep_wait();
  const uint32_t tmem = *tmem_slot;
  const int items = p.row_tiles * p.shares;
  const int blocks = (p.K + kBlockK - 1) / kBlockK;
  const int item0 = blockIdx.x / CTAS, step = gridDim.x / CTAS;

  if (warp == 0) {
    // The whole warp walks the loop, one thread issues: with `lane == 0` around the loops of both
    // warps a K block took 0.43 us however little it held, so 0.33 (700 rows x 3,000 tokens, K =
    // 2,000: 23.3 and 20.7 us).
    const bool one = elect_one();
    const uint64_t once = policy_evict_first();  // with one row tile, w only passes through L2
    int s = 0, it = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (int item = item0; ok && item < items; item += step) {
      int u0, u1;
      share_units(p, item / p.row_tiles, u0, u1);
      const int row = ((item % p.row_tiles) * CTAS + rank) * kRows;
      for (int n; ok && u0 < u1; u0 += n) {
        n = next_tile<kTile>(u1 - u0);
        const int col = u0 * kUnit + rank * n * kBox;  // a pair splits the tile's rows of w
        for (int kb = 0; kb < blocks; kb += PER) {
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], phase, s_err, p.err, kErrWaitTimeoutProducer));
          if (!ok) break;
          if (one) {
            const int end = PER == 1 ? kb + 1 : min(kb + PER, blocks);
            if (rank == 0) mbar_arrive_expect_tx(&full[s], (end - kb) * CTAS * (p.x_bytes + n * kBoxBytes));
            uint8_t* at = smem + s * stage_bytes;
            const uint32_t bar = CTAS == 2 ? mapa_shared(smem_u32(&full[s]), 0) : 0;
#pragma unroll
            for (int b = kb; b < kb + PER; ++b, at += p.block_bytes) {
              if (PER > 1 && b >= end) break;
              if (CTAS == 2) {
                tma_load_2d_pair(at, &tmX, bar, b * kBlockK, row);
                for (int i = 0; i < n; ++i)
                  tma_load_2d_pair(at + p.x_bytes + i * kBoxBytes, &tmW, bar, b * kBlockK, col + i * kBox);
              } else {
                tma_load_2d(at, &tmX, &full[s], b * kBlockK, row);
                for (int i = 0; i < n; ++i) {
                  uint8_t* box = at + p.x_bytes + i * kBoxBytes;
                  if (p.row_tiles == 1) tma_load_2d_hint(box, &tmW, &full[s], b * kBlockK, col + i * kBox, once);
                  else tma_load_2d(box, &tmW, &full[s], b * kBlockK, col + i * kBox);
                }
              }
            }
          }
          ++it;
          if (++s == stages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
    }
    // loads in flight land before the CTA gives up its memory (a pair's count on its first CTA)
    if (rank == 0)
      for (int j = max(0, it - stages); j < it && !ok; ++j) mbar_drain(&full[j % stages], (j / stages) & 1);
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const bool one = elect_one();
      const uint64_t a0 = sdesc_kmajor_sw128(smem_u32(smem));
      int s = 0, tc = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int item = item0; ok && item < items; item += step) {
        int u0, u1;
        share_units(p, item / p.row_tiles, u0, u1);
        for (int n; ok && u0 < u1; u0 += n) {
          n = next_tile<kTile>(u1 - u0);
          const uint32_t idesc = idesc_bf16_f32(CTAS * kRows, n * kUnit);
          for (int kb = 0; kb < blocks; kb += PER) {
            const int buf = tc & 1;
            if (kb % SEG == 0)
              ok = __all_sync(0xffffffffu, mbar_wait(&tempty[buf], ((tc >> 1) & 1) ^ 1, s_err, p.err, kErrWaitTimeoutMma));
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&full[s], phase, s_err, p.err, kErrWaitTimeoutMma));
            if (!ok) break;
            tc_fence_after();
            const uint64_t a = a0 + uint32_t(s * (stage_bytes >> 4)), b = a + (p.x_bytes >> 4);
            const uint32_t block = p.block_bytes >> 4;
            const bool last = (kb + PER) % SEG == 0 || kb + PER >= blocks;
            if (one) {
#pragma unroll
              for (int j = 0; j < PER; ++j) {
                if (j > 0 && kb + j >= blocks) break;
#pragma unroll
                for (int k = 0; k < kBlockK / 16; ++k) {
                  const uint32_t more = (kb % SEG > 0 || j + k > 0) ? 1u : 0u;
                  if (CTAS == 2) umma_f16_pair(tmem + buf * kCols, a + j * block + 2 * k, b + j * block + 2 * k, idesc, more);
                  else umma_f16(tmem + buf * kCols, a + j * block + 2 * k, b + j * block + 2 * k, idesc, more);
                }
              }
              if (CTAS == 2) {
                umma_commit_pair(&empty[s]);
                if (last) umma_commit_pair(&tfull[buf]);
              } else {
                umma_commit(&empty[s]);
                if (last) umma_commit(&tfull[buf]);
              }
            }
            __syncwarp();
            if (last) ++tc;
            if (++s == stages) {
              s = 0;
              phase ^= 1;
            }
          }
        }
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const int m = q * 32 + lane;
    const uint32_t mine = tmem + (uint32_t(q * 32) << 16) + half * kHalf;
    int tc = 0;
    bool ok = true;
    for (int item = item0; item < items; item += step) {
      const int share = item / p.row_tiles;
      int u0, u1;
      share_units(p, share, u0, u1);
      const int row = ((item % p.row_tiles) * CTAS + rank) * kRows + m;
      const int id = row < p.T ? p.ids[row] : -1;
      LogprobSums a;
      float given = 0.f;
      for (int n; ok && u0 < u1; u0 += n) {
        n = next_tile<kTile>(u1 - u0);
        const int first = u0 * kUnit + half * kHalf;
        // columns of this thread: up to the tile's end and the vocabulary's
        const int cols = min(kHalf, min((u0 + n) * kUnit, p.V) - first);
        float v[kHalf];
        for (int kb = 0; ok && kb < blocks; kb += SEG, ++tc) {
          const int buf = tc & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&tfull[buf], (tc >> 1) & 1, s_err, p.err, kErrWaitTimeoutEpilogue));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kHalf; c += 32) {
            uint32_t r0[16], r1[16];
            tmem_ld16_issue(mine + buf * kCols + c, r0);
            tmem_ld16_issue(mine + buf * kCols + c + 16, r1);
            tmem_ld_wait(r0);
            tmem_ld_wait(r1);
            if (kb == 0) {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                v[c + j] = __uint_as_float(r0[j]);
                v[c + 16 + j] = __uint_as_float(r1[j]);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                v[c + j] += __uint_as_float(r0[j]);
                v[c + 16 + j] += __uint_as_float(r1[j]);
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CTAS == 2) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[buf]), 0));
            else mbar_arrive(&tempty[buf]);
          }
        }
        if (!ok || cols <= 0) continue;
        if (cols < kHalf) {
#pragma unroll
          for (int j = 0; j < kHalf; ++j)
            if (j >= cols) v[j] = -INFINITY;
        }
        const int want = id - first;
        if (__any_sync(0xffffffffu, want >= 0 && want < cols)) {
#pragma unroll
          for (int j = 0; j < kHalf; ++j)
            if (j == want && want < cols) given = v[j];
        }
        float top[4] = {v[0], v[1], v[2], v[3]};  // four chains of maxima, not one of 128
#pragma unroll
        for (int j = 4; j < kHalf; ++j) top[j & 3] = fmaxf(top[j & 3], v[j]);
        a.raise(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
        const float sh = a.shift();
        const u64t shift = pack2(sh, sh);
        u64t s0 = 0, s1 = 0, e0 = 0, e1 = 0;
#pragma unroll
        for (int j = 0; j < kHalf; j += 4) {
          logprob_terms<true>(v[j], v[j + 1], shift, s0, e0);
          logprob_terms<true>(v[j + 2], v[j + 3], shift, s1, e1);
        }
        float s, t, e, f;
        unpack2(add2(s0, s1), s, t);
        unpack2(add2(e0, e1), e, f);
        a.add_long(s + t, e + f);
      }
      if (!ok) a.hi = NAN;
      p.part[(long long)(share * 2 + half) * p.row_tiles * CTAS * kRows + row] = make_float4(a.m, a.hi + a.lo, a.e + a.el, given);
    }
  }
  if (CTAS == 2) cluster_sync();  // a pair's shared memory serves both CTAs
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if (CTAS == 2) tmem_dealloc_pair<2 * kCols>(tmem);
    else tmem_dealloc<2 * kCols>(tmem);
  }
}

// One warp per row joins its shares; a lane has all its parts under way before it uses one. A
// CTA is one warp: rows' scattered parts are read by as many SMs as there are rows (128 rows x
// 296 parts: 8.7 us with the kernel before it, 16.7 us with four warps to a CTA).
__global__ void __launch_bounds__(32) lm_logprobs_join_kernel(const float4* __restrict__ part, int parts, int pitch,
                                                               int T, int V, const int* __restrict__ ids,
                                                               float* __restrict__ lp, float* __restrict__ entropy) {
  constexpr int kAhead = 10;  // 320 parts at once: two for each of 148 CTAs
  griddep_wait();
  griddep_launch();
  const int row = blockIdx.x, lane = threadIdx.x & 31;
  if (row >= T) return;
  const int id = ids[row];
  float m = -INFINITY, given = 0.f;
  double s = 0.0, e = 0.0;
  for (int i0 = 0; i0 < parts; i0 += 32 * kAhead) {
    float4 t[kAhead];
    float top = m;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * 32 + lane;
      t[u] = i < parts ? part[(long long)i * pitch + row] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) top = fmaxf(top, t[u].x);
    top = warp_max(top);
    const float d0 = m == -INFINITY ? 0.f : fmaxf((m - top) * kLog2e, -300.f);
    const double f0 = fast_exp2(d0);
    e = f0 * (e + s * d0);
    s = f0 * s;
    m = top;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float d = t[u].x == -INFINITY ? 0.f : fmaxf((t[u].x - top) * kLog2e, -300.f);
      const float f = fast_exp2(d);
      s += f * t[u].y;
      e += f * fmaf(t[u].y, d, t[u].z);
      given += t[u].w;  // one share's, the others hold 0
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    e += __shfl_xor_sync(0xffffffffu, e, o);
    given += __shfl_xor_sync(0xffffffffu, given, o);
  }
  if (lane != 0) return;
  const bool bad = s != s, empty = !bad && s == 0.0;
  const float log_s = empty ? 0.f : s < 2.0 ? log1pf(float(s - 1.0)) : logf(float(s));
  entropy[row] = bad ? NAN : empty ? 0.f : float(log_s - e / s * kLn2);
  lp[row] = id == -1 ? 0.f : (id < 0 || id >= V || bad) ? NAN : (given - (empty ? 0.f : m)) - log_s;
}

// Clocks that a tile of `n` units keeps a CTA busy: per K block the most of what its warps need
// to issue (420 a pair, 600 a single CTA; less in stages of two blocks), the tensor core's two per column of logits, and its
// copies at 60 bytes a clock from L2; at least an epilogue's 2,500.
template <int CTAS>
static long long tile_clocks(int n, int x_rows, int blocks) {
  const int copies = (x_rows + n * kBox) * kBlockK * 2 / 60;
  return std::max<long long>(2500, (long long)blocks * std::max({CTAS == 2 ? 420 : 600, n * Lm<CTAS>::kUnit * 2, copies}));
}

// The vocabulary's shares per row tile are those that keep the busiest CTA the shortest time, but
// never shorter than the power limit leaves all of them, which over a longer while is two thirds
// of the tensor cores' clocks.
template <int CTAS>
static LmPlan plan_as(int T, int V, int K, int num_sms, long long& cost) {
  using C = Lm<CTAS>;
  LmPlan l;
  l.ctas = CTAS;
  l.row_tiles = (T + kRows * CTAS - 1) / (kRows * CTAS);
  l.units = (V + C::kUnit - 1) / C::kUnit;
  const int workers = std::max(1, num_sms / CTAS), blocks = (K + kBlockK - 1) / kBlockK;
  const long long power = (long long)l.row_tiles * CTAS * l.units * C::kUnit * 2 * blocks / num_sms * 3 / 2;
  long long clocks[C::kTile + 1];
  for (int n = 0; n <= C::kTile; ++n) clocks[n] = tile_clocks<CTAS>(n, std::min(T, kRows), blocks);
  constexpr long long kItemClocks = 5000;
  cost = -1;
  for (int rounds = (l.row_tiles + workers - 1) / workers;; ++rounds) {
    const int most = (int)std::min<long long>({(long long)rounds * workers / l.row_tiles, l.units, workers});
    const int of_share = (l.units + most - 1) / most, tiles = (of_share + C::kTile - 1) / C::kTile;
    const int n = of_share / tiles, more = of_share % tiles;  // `more` tiles have n + 1 units
    const long long busy = kItemClocks + (tiles - more) * clocks[n] + more * clocks[std::min(n + 1, C::kTile)];
    if (cost < 0 || rounds * busy < cost) {
      cost = rounds * busy;
      l.shares = (l.units + of_share - 1) / of_share;
      // No more shares than keep the busiest as long (10,007 tokens, 61 rows: 13.9 us in 79 shares of
      // two units, 16.0 in 148), unless a CTA's copies, x again for each tile, are what it waits
      // for: then all SMs help (102,400 tokens, 61 rows: 73 us in 148 shares, 78.5 in 146; 151,936
      // tokens, 128 rows: 105 in 148, 109 in 140, but 16 rows 106 in 148, 99 in 140).
      if (CTAS == 1 && l.row_tiles == 1 && T > 16 && of_share >= C::kTile) l.shares = most;
    }
    if (most == l.units || most == workers) break;
  }
  cost = std::max(cost, power);
  return l;
}

// CTA pairs read half as much of w per SM (8,192 x 102,400 x 2,048 2.27 ms in a short run, single CTAs on
// the same card 2.56; 256 x 32,000 x 4,096 67 us against 72, 512 x 10,007 x 1,000 23 against 26), single CTAs' items
// are finer and the last row tile's empty rows fewer (333 x 10,007 x 1,000 19 us, pairs 21; 300 x
// 50,000 x 2,048 71 against 80). One row tile stays on single CTAs and their short segments.
static LmPlan best_shares(int T, int V, int K, int num_sms) {
  long long one = 0, two = 0;
  const LmPlan single = plan_as<1>(T, V, K, num_sms, one);
  if (T <= kRows || num_sms < 2) return single;
  const LmPlan pairs = plan_as<2>(T, V, K, num_sms, two);
  return two <= one ? pairs : single;
}

// Rows of a box of x. A few rows load only themselves (in swizzle atoms of 8): a CTA's copies move
// about 55 GB/s in rows of 128 bytes, and x, read again for each tile, should not take a third of it.
// The MMA's other rows are whatever shared memory held; theirs are results that nobody reads.
static int x_rows(const LmPlan& l, int T) { return l.row_tiles * l.ctas == 1 ? (T + 7) / 8 * 8 : kRows; }
static int block_bytes(const LmPlan& l, int T) {  // of x and of the boxes of the largest tile
  const int boxes = std::min(kCols / (kBox * l.ctas), (l.units + l.shares - 1) / l.shares);
  return x_rows(l, T) * kBlockK * 2 + boxes * kBoxBytes;
}

LmPlan lm_plan(int T, int V, int K, int num_sms) {
  LmPlan l = best_shares(T, V, K, num_sms);
  const bool many = l.ctas == 2 && V >= kManyTokens;
  l.segment = many ? 16 : l.row_tiles > 1 || l.ctas == 2 ? 8 : 4;
  // Stages of two K blocks where four fit: a narrow share's K block costs what its warps need to
  // issue it, half of which is the stage's (9,472 tokens, 16 rows: 0.33 us a block, in twos 0.26).
  // Single CTAs on several row tiles hold 128 rows of x and shares that are too wide for that.
  l.per_stage = (l.ctas == 2 ? !many : l.segment == 4) && 8 * block_bytes(l, T) <= kRing ? 2 : 1;
  return l;
}

template <int CTAS, int SEG, int PER>
static void launch_lm(const LmPlan& l, const CUtensorMap& tx, const CUtensorMap& tw, const LmParams& p, int num_sms,
               cudaStream_t s) {
  auto kern = lm_logprobs_kernel<CTAS, SEG, PER>;
  set_smem_bytes(kern, kSmem);
  prefer_max_smem_carveout(reinterpret_cast<const void*>(kern));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attrs[2];
  cfg.gridDim = dim3(CTAS * (unsigned)std::min<long long>(num_sms / CTAS, (long long)l.row_tiles * l.shares));
  cfg.blockDim = dim3(64 + kEpilogue);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cfg.attrs = attrs;
  if (CTAS == 2) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attrs[cfg.numAttrs].val.clusterDim.x = 2;
    attrs[cfg.numAttrs].val.clusterDim.y = 1;
    attrs[cfg.numAttrs].val.clusterDim.z = 1;
    cfg.numAttrs += 1;
  }
  if (pdl_enabled()) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs += 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tx, tw, p);
  if (e != cudaSuccess) throw std::runtime_error(std::string("lm_logprobs launch failed: ") + cudaGetErrorString(e));
}

void lm_logprobs(const LmPlan& l, const void* x, long long ldx, const void* w, long long ldw, int T, int V, int K,
                 const int* ids, void* workspace, float* lp, float* entropy, int* err, int num_sms, cudaStream_t s) {
  if (T <= 0) return;
  LmParams p = {};
  p.T = T;
  p.V = V;
  p.K = K;
  p.row_tiles = l.row_tiles;
  p.units = l.units;
  p.shares = l.shares;
  p.ids = ids;
  p.part = static_cast<float4*>(workspace);
  p.err = err;
  p.x_bytes = x_rows(l, T) * kBlockK * 2;
  p.block_bytes = block_bytes(l, T);
  const int per = l.per_stage;
  p.stage_bytes = per * p.block_bytes;
  // the MMA reads 128 rows of x from the last block too, whatever a box holds
  const int behind = (per - 1) * p.block_bytes + std::max(p.block_bytes, kXBytes);
  p.stages = std::min(kMaxStages, (kRing - behind) / p.stage_bytes + 1);
  CUtensorMap tx, tw;
  make_tmap_2d(&tx, x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, T, K, ldx, x_rows(l, T), kBlockK);
  make_tmap_2d(&tw, w, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, V, K, ldw, kBox, kBlockK);
  if (l.segment == 16) launch_lm<2, 16, 1>(l, tx, tw, p, num_sms, s);
  else if (l.ctas == 2) per == 2 ? launch_lm<2, 8, 2>(l, tx, tw, p, num_sms, s) : launch_lm<2, 8, 1>(l, tx, tw, p, num_sms, s);
  else if (l.segment == 8) launch_lm<1, 8, 1>(l, tx, tw, p, num_sms, s);
  else per == 2 ? launch_lm<1, 4, 2>(l, tx, tw, p, num_sms, s) : launch_lm<1, 4, 1>(l, tx, tw, p, num_sms, s);
  launch_k(lm_logprobs_join_kernel, dim3(T), dim3(32), 0, s, (const float4*)workspace, 2 * p.shares,
           p.row_tiles * l.ctas * kRows, T, V, ids, lp, entropy);
}

}  // namespace sp
