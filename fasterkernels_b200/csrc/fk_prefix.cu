// fk_prefix.cu -- decode attention of a batch whose sequences share a prefix.
//
// Sequence b attends the prefix's P tokens and then its own.  Softmax
// statistics join by log-sum-exp, so the two parts are computed apart: the
// prefix once for the whole batch (below), the own tokens by the split-KV
// decode kernel (fk_decode_kernel.cuh), which leaves its segments' (max, sum,
// acc) in the workspace; a last kernel joins them all with the sink.
//
// Prefix part.  For one KV head the batch's query heads are the rows of a
// matrix: row r = b * G + g, R = B * G rows, and the work is S = Q K^T (R x P),
// a softmax numerator per row and O = P V.  Reading the prefix once for up to
// 256 rows turns a read of B x P tokens into a matrix product of 4 R P D
// operations per KV head on 2 P D elements: tensor cores, not memory, carry it
// from about 256 rows on.
//
//   tcgen05 tiles of 128 rows x 64 tokens.  Two independent streams, each with
//   a warpgroup of softmax threads (thread = row), take turns on the tensor
//   cores; with more than 128 rows they are two row tiles that share each K / V
//   tile (dual), otherwise the two halves of each token tile (parity).  Tensor
//   memory holds for each stream O (f32, D columns) and two items of S (f32, 64
//   columns each): S of item j + 1 is there before the softmax of item j ends,
//   so that it never waits for the chain P V, Q K^T.  (With 128-token items there
//   is room for one S a stream, and that chain, 1100 cycles, was added to every
//   tile: 395 us instead of 319, at that time, for the long case below.)  P (f16, or bf16 for bf16 KV)
//   overwrites half of its own S and is the A operand of O += P V from there:
//   the type that V has or is widened to, since the tensor cores take A and B of
//   one 16-bit type (f32 P would be a second product for its low half).  That
//   rounding is of the size of the output's own, so errors are 1.1 to 1.4 times
//   those of 32-bit P; the sum of P is of the unrounded ones, in 32 bits.
//
// Work is cut like the decode kernel's: units (KV head, one or two row tiles)
// laid end to end in granules (dual: one token tile, parity: two), each CTA of
// the persistent grid takes an equal run of them, and the piece of a unit in a
// CTA is a segment whose (max, sum, O) goes to the workspace.  Planned on the
// device from the prefix length and the own lengths.
//
// Warps: 0-3 and 4-7 softmax of stream 0 and 1 (they load Q too), 8-11 load K
// and V, 12 issues the MMAs.  A tile that the tensor cores read with one
// descriptor needs its 8-row groups evenly spaced, so a page is loaded as one
// box per 128-byte half, straight into its 16 rows of that half.  Each loader
// warp loads two of a tile's eight pages: one warp issues a box in 100 to 150
// cycles, and a tile's K and V are 32 boxes for 1024 to 2048 cycles of tensor
// work.  e4m3 pages land in a ring of the warp's own and are widened to f16
// from there.  Tiles that end the prefix or hold a bad page are loaded row by
// row instead, with zeros where there is no token (the tail of a page may hold
// anything, and 0 x NaN would reach the output).
//
// Bound.  An item pair takes 1280 cycles of tensor work: Q K^T with N = 64 runs
// at the rate of its shared-memory reads (48 cycles per MMA of 32: 4 KB of Q and 2
// KB of K at 128 bytes a cycle), P V at the MMA rate.  Measured 1800 to 1950
// cycles: the chain P ready -> P V, Q K^T issue -> S ready passes through one
// issuing warp, and e4m3 widening takes 512 cycles of shared-memory bandwidth more.
// Device times, own part and join included (B200): long case, 128 sequences x 64
// heads (8 KV heads), 65536 tokens of e4m3 + tails up to 1000, 303 us = 0.92
// PFLOP/s; 64 x 32 heads, 32768 tokens of f16 + tails up to 512, 71 us, of which
// the own part's reads take 20 to 27 and the join 9; 2 x 32 heads, 131072 tokens of
// bf16, 108 us = 5.0 TB/s; 4 x 32 heads, 1000 tokens, 17 us, three kernels'
// latencies.
#include <cuda_fp8.h>

#include <atomic>
#include <chrono>
#include <type_traits>

#include "fk_decode_kernel.cuh"
#include "fk_host.h"
#include "fk_prefix.h"
#include "fk_tc.cuh"

namespace fk {

constexpr int SOFT_WARPS = 8;  // warps 0-7: softmax; 8-11 loaders; 12 MMA issue
constexpr int LOAD_WARP = SOFT_WARPS, MMA_WARP = SOFT_WARPS + 4;
constexpr int PTHREADS = (MMA_WARP + 1) * 32;
constexpr int PROWS = 128;    // rows of a row tile (MMA M)
constexpr int PTOK = 128;     // tokens of a token tile (a K or V tile in shared memory)
constexpr int PITEM = 64;     // tokens of an item (MMA N of QK, K of PV): half a tile
constexpr int PPAGES = PTOK / PAGE;
constexpr int HALF_BYTES = PTOK * 128;  // 128 rows of a 128-byte half
// Of eight pairs of exponentials, those computed on the FMA units: measured 0:
// 305 us, 1: 301, 2: 304 for the long case below, equal for the others.
constexpr int FMA_PAIRS = 1;
// Granules that starting behind the own part costs a CTA.  16-bit, 32 x 8 heads,
// 4096 tokens behind 16 tails of 20: 17.4 us with 64 CTAs of two granules, 23.2
// with 128 of one, which the SMs beside the own part do not hold.  2 to 9
// measured: from 4 on some calls lose (48 x 64 heads, 2048 tokens: 30 -> 43 us).
constexpr int WAIT = 2;

template <int KV, int D>
struct PCfg {
  static constexpr bool FP8 = KV == FK_DTYPE_E4M3;
  static constexpr int NH = D / 64;
  static constexpr int TILE_BYTES = NH * HALF_BYTES;  // Q, K or V tile in 16 bits
  static constexpr int STAGES = D == 64 ? 8 : FP8 ? 4 : 5;
  static constexpr int RAW = FP8 ? 2 : 0;             // e4m3 tiles on the way
  static constexpr int TILES = (2 + STAGES) * TILE_BYTES + RAW * HALF_BYTES;
};

// Barriers and small exchanges, behind the tiles.
template <int ST, int RAW>
struct PShared {
  uint64_t full[ST], empty[ST], qfull, qempty, s[2][2], p[2][2], o[2], done[2], drain;
  uint64_t raw[4][RAW];              // a loader warp's e4m3 pages
  uint32_t tmem;
  int busy;                          // SMs at work on the own part
  volatile int bad;                  // a bad page was seen: the softmax checks pages from then on
};
template <int KV, int D>
constexpr int prefix_smem() {
  using C = PCfg<KV, D>;
  return C::TILES + static_cast<int>(sizeof(PShared<C::STAGES, C::RAW ? C::RAW : 1>));
}
static_assert(prefix_smem<FK_DTYPE_F16, 128>() <= 227 * 1024 && prefix_smem<FK_DTYPE_E4M3, 128>() <= 227 * 1024,
              "shared memory of a block");

struct PrefixParams {
  CUtensorMap tk, tv;  // boxes of one page's 16 rows x 128 bytes
  const void* q;
  long long q_b, q_h;
  const void* k;
  const void* v;
  long long kp_p, kp_h, kp_s, vp_p, vp_h, vp_s;
  const int* table;     // prefix pages
  const int* plen_dev;  // prefix length on the device, or null: plen
  int plen, blocks, num_pages;
  int rows, G, kv_heads, q_dtype, q_al16;
  const float* scale_q;
  const float* scale_k;
  const int* seq_lens;  // of the own tokens: what keeps SMs from the prefix at first
  int batch, own_items;
  int* plan;            // granules of a CTA, for the join
  const unsigned long long* ticket;  // the own part's word, and what it is set to
  unsigned long long ticket_value;
  float2* ml;
  float* acc;
  int* status;          // or null
  unsigned long long wait_ns;
  int inject;
};

// Granules and units, from the prefix length (device side).  In 32 bits: the
// host refuses more than 2^30 granules.
struct PrefixPlan {
  int nt, nd, upu;       // token tiles; dual units and units of a KV head
  int gh, total;         // granules of a KV head, in all
  int per;               // of a CTA
  __device__ PrefixPlan(int plen, int rows, int kv_heads) {
    const int rt = (rows + PROWS - 1) / PROWS;
    nt = (plen + PTOK - 1) / PTOK;
    nd = rt / 2;
    upu = nd + (rt & 1);
    gh = nd * nt + ((rt & 1) ? (nt + 1) / 2 : 0);
    total = gh * kv_heads;
  }
  // A CTA that finds its SM taken by the own part starts about as late as
  // WAIT granules take, so with few granules a run that fits the other SMs'
  // CTAs is the shorter way.
  __device__ void cut(int ctas, int busy) {
    per = max((total + ctas - 1) / ctas, 1);
    if (ctas > busy) {
      const int few = (total + ctas - busy - 1) / (ctas - busy);
      if (few - per <= WAIT) per = max(few, 1);
    }
  }
  // First granule and length of unit u of a KV head.
  __device__ int unit_base(int u) const { return u * nt; }
  __device__ int unit_len(int u) const { return u < nd ? nt : (nt + 1) / 2; }
};

// The prefix's length: at most what its table holds (tokens past that are
// masked like those of a bad page).
__device__ __forceinline__ int prefix_len(const int* dev, int host, int blocks, bool* past) {
  const int n = max(dev != nullptr ? __ldg(dev) : host, 0);
  *past = n > blocks * PAGE;
  return min(n, blocks * PAGE);
}

struct PrefixSeg {
  int h, unit, seg, dual, t0, tiles;  // token tiles [t0, t0 + tiles)
};

// The segment at granule g of CTA c (granules [.., end)); returns its length.
__device__ __forceinline__ int prefix_segment(const PrefixPlan& pl, int g, int end, int c, PrefixSeg* s) {
  s->h = g / pl.gh;
  const int r = g - s->h * pl.gh;
  s->dual = r < pl.nd * pl.nt;
  s->unit = s->dual ? r / pl.nt : pl.nd;
  const int off = r - pl.unit_base(s->unit);
  const int n = min(end - g, pl.unit_len(s->unit) - off);
  s->seg = c + s->h * pl.upu + s->unit;
  s->t0 = s->dual ? off : 2 * off;
  s->tiles = s->dual ? n : min(2 * n, pl.nt - 2 * off);
  return n;
}

// Load order of a segment of m token tiles: dual K0 V0 K1 V1 ..; parity K0 K1
// V0 K2 V1 K3 .. V(m-2) V(m-1).  It is the order in which the tiles are used.
__device__ __forceinline__ int load_item(int idx, int m, int dual, bool* is_v) {
  if (dual || m == 1) {
    *is_v = idx & 1;
    return idx >> 1;
  }
  if (idx < 2) {
    *is_v = false;
    return idx;
  }
  const int j = idx - 2;
  if (j < 2 * (m - 2)) {
    *is_v = !(j & 1);
    return (j >> 1) + ((j & 1) ? 2 : 0);
  }
  *is_v = true;
  return j - (m - 2);
}

// Eight consecutive Q elements as packed pairs of the MMA type.
template <bool MBF16>
__device__ __forceinline__ uint4 load_q8(const PrefixParams& p, long long e, float sq, uint32_t flip) {
  uint32_t w[4];
  if (p.q_dtype == FK_DTYPE_E4M3) {
    const unsigned char* src = static_cast<const unsigned char*>(p.q) + e;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t raw = __ldg(reinterpret_cast<const unsigned short*>(src) + i);
      const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(raw), __NV_E4M3)));
      w[i] = pack2<MBF16>(f.x * sq, f.y * sq);
    }
  } else {
    const unsigned short* src = static_cast<const unsigned short*>(p.q) + e;
    if (p.q_al16) {
      const uint4 r = __ldg(reinterpret_cast<const uint4*>(src));
      w[0] = r.x;
      w[1] = r.y;
      w[2] = r.z;
      w[3] = r.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(src) + i);
    }
    if (!MBF16 && p.q_dtype == FK_DTYPE_BF16) {  // bf16 Q over e4m3 KV
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack2<false>(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
  return make_uint4(w[0] ^ flip, w[1] ^ flip, w[2] ^ flip, w[3] ^ flip);
}

template <int KV, int D>
__global__ void __launch_bounds__(PTHREADS, 1) prefix_kernel(const __grid_constant__ PrefixParams p) {
  using C = PCfg<KV, D>;
  constexpr bool FP8 = KV == FK_DTYPE_E4M3;
  constexpr bool MBF16 = KV == FK_DTYPE_BF16;
  constexpr int ST = C::STAGES;
  // f16 P is stored times 2^BIAS: with at most 2^8 above the reference maximum
  // it stays below 2^15, and the smallest P that does not vanish is 2^-32 of the
  // maximum's instead of 2^-25 (bf16 has f32's range and needs none).
  constexpr float BIAS = MBF16 ? 0.f : 7.f;
  constexpr float LAZY = 8.f;
  extern __shared__ __align__(1024) unsigned char smem_raw[];  // 1024: the swizzle's period
  const uint32_t sQ = smem_u32(smem_raw);             // [2] row tiles
  const uint32_t sKV = sQ + 2 * C::TILE_BYTES;        // [ST]
  const uint32_t sRaw = sKV + ST * C::TILE_BYTES;     // [RAW][loader warp] two e4m3 pages
  constexpr int RAW = C::RAW > 0 ? C::RAW : 1;
  PShared<ST, RAW>& sh = *reinterpret_cast<PShared<ST, RAW>*>(smem_raw + C::TILES);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == 1 && lane == 0) {  // not a loader: what follows the fetch in its warp waits for it
    prefetch_tmap(&p.tk);
    prefetch_tmap(&p.tv);
  }
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(smem_u32(&sh.full[i]), 4);
      mbar_init(smem_u32(&sh.empty[i]), 1);
    }
    mbar_init(smem_u32(&sh.qfull), SOFT_WARPS);
    mbar_init(smem_u32(&sh.qempty), 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&sh.s[0][0] + i), 1);
      mbar_init(smem_u32(&sh.p[0][0] + i), 4);
    }
    mbar_init(smem_u32(&sh.o[0]), 1);
    mbar_init(smem_u32(&sh.o[1]), 1);
    mbar_init(smem_u32(&sh.done[0]), 1);
    mbar_init(smem_u32(&sh.done[1]), 1);
    mbar_init(smem_u32(&sh.drain), 1);
    for (int i = 0; i < 4 * RAW; ++i) mbar_init(smem_u32(&sh.raw[0][0] + i), 1);
    fence_mbar_init();
    sh.bad = 0;
  }
  if (warp == MMA_WARP) tmem_alloc(smem_u32(&sh.tmem), 512);
  // The kernel before this one in the stream is the own part's, which this one
  // does not depend on: its blocks start as SMs come free and only wait for it
  // before they end (so that the join, which waits for this kernel, finds both
  // parts).  Waiting for it here instead costs 4 to 11 us a call (4 x 32 heads,
  // 1000 tokens: 23.5 us instead of 16.6).  What both read was written before the
  // own part's wait returned; its ticket, released after that wait and acquired
  // here (0.2 to 0.4 us), is what makes those writes this kernel's to see.  Its
  // blocks start this kernel later than that, so the ticket is there; if not,
  // this kernel waits too.
  if (tid == 96 && ld_acquire_gpu(p.ticket) != p.ticket_value) grid_dependency_wait();
  __syncthreads();
  bool past;
  const int plen = prefix_len(p.plen_dev, p.plen, p.blocks, &past);
  if (warp == 2) {
    // SMs that the own part keeps busy, by its plan: equal runs of 16-token
    // granules, MIN_PER at least, over its grid, whose CTAs go to SMs of their
    // own first.  Only whether all are busy counts, so a prefix of the batch may do.
    long long u = 0;
    const long long all = static_cast<long long>(gridDim.x) * MIN_PER;
    for (int b0 = 0; b0 < p.batch && u < all; b0 += 128) {
      long long n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int b = b0 + 32 * i + lane;
        if (b < p.batch) n += (max(__ldg(p.seq_lens + b), 0) + 15ll) >> 4;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      u += n * p.own_items;
    }
    if (lane == 0) sh.busy = static_cast<int>(min((u + MIN_PER - 1) / MIN_PER, static_cast<long long>(gridDim.x)));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = 0;  // all 512 columns are ours, so the allocation starts at column 0
  grid_dependency_trigger();

  if (past && blockIdx.x == 0 && tid == 0 && p.status != nullptr) atomicOr(p.status, FK_STATUS_BAD_PAGE);
  PrefixPlan pl(plen, p.rows, p.kv_heads);
  pl.cut(gridDim.x, sh.busy);
  if (blockIdx.x == 0 && tid == 0) *p.plan = pl.per;
  const int g0 = min(static_cast<int>(blockIdx.x) * pl.per, pl.total), g1 = min(g0 + pl.per, pl.total);
  const float sk = (FP8 && p.scale_k != nullptr) ? __ldg(p.scale_k) : 1.f;
  auto timed_out = [&]() {
    if (lane == 0 && p.status != nullptr) atomicOr(p.status, FK_STATUS_TIMEOUT);
  };
  // Whole-warp wait; false (for every lane) when it ran out.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    const bool ok = mbar_wait(smem_u32(bar), parity, p.wait_ns);
    if (__all_sync(0xffffffffu, ok)) return true;
    timed_out();
    return false;
  };

  if (warp < SOFT_WARPS) {
    // ============================================================ softmax
    const int s = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // lane (warp & 3) * 32 in bits 16..
    const uint32_t tO = tmem + lanes + 256 + s * D;
    // never 0: a masked logit (-inf) stays one (and NaN stays NaN)
    const float cs = rsqrtf(static_cast<float>(D)) * LOG2E * fabsf(sk);
    const float c = cs < 1e-30f ? 1e-30f : cs;
    uint32_t sph = 0;  // parities of the two S buffers
    uint32_t oph = 0, dph = 0;  // parities of o (segments of more than one item) and done
    uint32_t qph = 1;
    const float sq = p.scale_q != nullptr ? __ldg(p.scale_q) : 1.f;
    const uint32_t flip = sk < 0.f ? 0x80008000u : 0u;  // a negative scale turns Q over: the softmax sees |scale|
    bool alive = true;
    for (int g = g0; g < g1 && alive;) {
      PrefixSeg sg;
      g += prefix_segment(pl, g, g1, blockIdx.x, &sg);
      const int ni = sg.dual ? 2 * sg.tiles : sg.tiles;
      const int trow = (2 * sg.unit + (sg.dual ? s : 0)) * PROWS + row;
      const int tok00 = sg.t0 * PTOK + (sg.dual ? 0 : s * PITEM), tstep = sg.dual ? PITEM : PTOK;
      // ---- Q: this stream's row tile (parity: the one tile, by stream 0), once
      // the previous segment's products are done.  The softmax threads have
      // nothing else to do yet, while a loader waits 2000 to 5000 cycles behind
      // its first TMA (the tensor map is fetched then).
      if (!(alive = wait(&sh.qempty, qph))) break;
      qph ^= 1u;
      if (sg.dual || s == 0) {
        // Q of the MMA's type with aligned rows: all loads of the tile in flight
        const bool q_plain = p.q_al16 != 0 && p.q_dtype == (MBF16 ? FK_DTYPE_BF16 : FK_DTYPE_F16) && flip == 0;
        constexpr int CPR = D / 8, RPS = 128 / CPR;  // 16-byte chunks of a row, rows of a step
        static_assert(RPS % 8 == 0, "the swizzle of row r0 + k RPS is that of row r0");
        const int lt = tid & 127, ch = lt % CPR, r0 = lt / CPR;
        // rows r0, r0 + RPS, ..: their element offsets go up by one step, and by
        // one turn more where the step passes the end of a group
        const int db = RPS / p.G, dg = RPS - db * p.G;
        const long long step = db * p.q_b + dg * p.q_h, turn = p.q_b - p.G * p.q_h;
        const int first = (2 * sg.unit + (sg.dual ? s : 0)) * PROWS + r0;
        const int b = first / p.G;
        int gg = first - b * p.G, left = p.rows - first;
        long long e = b * p.q_b + (sg.h * p.G + gg) * p.q_h + ch * 8;
        const uint32_t dst = sQ + s * C::TILE_BYTES + (ch >> 3) * HALF_BYTES + r0 * 128 +
                             (static_cast<uint32_t>((ch & 7) ^ (r0 & 7)) << 4);
        auto advance_row = [&]() {
          left -= RPS;
          e += step;
          if ((gg += dg) >= p.G) {
            gg -= p.G;
            e += turn;
          }
        };
        const uint4 none = make_uint4(0u, 0u, 0u, 0u);
        if (q_plain) {
          uint4 x[PROWS / RPS];
#pragma unroll
          for (int k = 0; k < PROWS / RPS; ++k, advance_row()) {
            x[k] = none;
            if (left > 0) x[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p.q) + e));
          }
#pragma unroll
          for (int k = 0; k < PROWS / RPS; ++k) sts128(dst + k * RPS * 128, x[k].x, x[k].y, x[k].z, x[k].w);
        } else {
#pragma unroll 1
          for (int k0 = 0; k0 < PROWS / RPS; k0 += 4) {
            uint4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k, advance_row()) x[k] = left > 0 ? load_q8<MBF16>(p, e, sq, flip) : none;
#pragma unroll
            for (int k = 0; k < 4; ++k) sts128(dst + (k0 + k) * RPS * 128, x[k].x, x[k].y, x[k].z, x[k].w);
          }
        }
        fence_async_proxy();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.qfull));
      float m = NEG_INF, l = 0.f;
      for (int j = 0; j < ni; ++j) {
        const int buf = j & 1;
        const int tok0 = tok00 + j * tstep;  // the item's first token
        const uint32_t tS = tmem + lanes + s * 128 + buf * PITEM;
        if (!(alive = wait(&sh.s[s][buf], (sph >> buf) & 1u))) break;
        sph ^= 1u << buf;
        tc_fence_after();
        // ---- the row of S, its maximum
        uint32_t r[2][32];
        tmem_ld32(tS, r[0]);
        tmem_ld32(tS + 32, r[1]);
        const int lim = plen - tok0;  // tokens of the item that exist
        uint32_t okp = 0xfu;          // its pages that do
        if (sh.bad) {
          okp = 0;
          for (int k = 0; k < PITEM / PAGE; ++k) {
            const int pg = tok0 / PAGE + k;
            const int ph = pg < p.blocks ? __ldg(p.table + pg) : -1;
            okp |= (ph >= 0 && ph < p.num_pages ? 1u : 0u) << k;
          }
        }
        tmem_wait_ld(r[0]);
        tmem_wait_ld(r[1]);
        if (lim < PITEM || okp != 0xfu) {
#pragma unroll
          for (int k = 0; k < PITEM; ++k)
            if (k >= lim || !((okp >> (k >> 4)) & 1u)) r[k >> 5][k & 31] = __float_as_uint(NEG_INF);
        }
        float mx0 = NEG_INF, mx1 = NEG_INF, mx2 = NEG_INF, mx3 = NEG_INF;
#pragma unroll
        for (int k = 0; k < PITEM; k += 8) {
          const uint32_t* q = &r[k >> 5][k & 31];
          mx0 = max3_nan(mx0, __uint_as_float(q[0]), __uint_as_float(q[1]));
          mx1 = max3_nan(mx1, __uint_as_float(q[2]), __uint_as_float(q[3]));
          mx2 = max3_nan(mx2, __uint_as_float(q[4]), __uint_as_float(q[5]));
          mx3 = max3_nan(mx3, __uint_as_float(q[6]), __uint_as_float(q[7]));
        }
        const float mx = max3_nan(max3_nan(mx0, mx1, mx2), mx3, mx3) * c;
        // The reference maximum moves only when a logit exceeds it by more than
        // LAZY (log2 units): any reference gives the same softmax once O and l
        // are normalised together, and O is rescaled in the first items only.
        // A NaN logit makes the reference, and so the whole row, NaN.
        const bool grow = !(mx <= m + LAZY);
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = grow ? mx : m;
          const float al = (m == NEG_INF) ? 0.f : ex2(m - mn);
          l *= al;
          if (j > 0) {
            // The previous item's P V is complete once S of the next item is,
            // which was issued behind it (no more than looked at here); the last
            // item has no next one, o[s] stands in for it.
            if (!(alive = j + 1 < ni ? wait(&sh.s[s][buf ^ 1], (sph >> (buf ^ 1)) & 1u) : wait(&sh.o[s], oph))) break;
            tc_fence_after();
            uint32_t o[16];
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
              tmem_ld16(tO + d, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * al);
              tmem_st16(tO + d, o);
            }
          }
          m = mn;
        }
        const float mb = (m == NEG_INF ? 0.f : m) - BIAS;
        // ---- P = 2^(x - m + BIAS).  Special-function units give 16 exponentials
        // a cycle and SM, as many as the tensor cores take; one pair of eight is
        // computed on the FMA units instead.
        const f2 c2 = mk2(c, c), mb2 = mk2(-mb, -mb);
        f2 l0 = mk2(0.f, 0.f), l1 = mk2(0.f, 0.f);
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            f2 x = fma2(mk2(__uint_as_float(r[ch][2 * k]), __uint_as_float(r[ch][2 * k + 1])), c2, mb2);
            float p0, p1;
            if (k % 8 < FMA_PAIRS) {
              x = exp2_fma(x);
              split2(x, p0, p1);
            } else {
              split2(x, p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
              x = mk2(p0, p1);
            }
            if (k & 1) l1 = add2(l1, x);
            else l0 = add2(l0, x);
            w[k] = pack2<MBF16>(p0, p1);
          }
          tmem_st16(tS + 16 * ch, w);  // over S, which is in registers
        }
        {
          float s0, s1;
          split2(add2(l0, l1), s0, s1);
          l += s0 + s1;
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.p[s][buf]));
      }
      if (!alive) break;
      if (ni > 1) oph ^= 1u;
      const long long rec = static_cast<long long>(sg.seg) * 2 + s;
      // the last P V
      if (!(alive = wait(&sh.done[s], dph))) break;
      dph ^= 1u;
      tc_fence_after();
      const bool valid = trow < p.rows;
      if (valid) p.ml[rec * PROWS + row] = make_float2(m == NEG_INF ? NEG_INF : m - BIAS, l);
      // [D / 4][128 rows][4]: a warp stores 512 contiguous bytes
      float4* dst = reinterpret_cast<float4*>(p.acc + rec * PROWS * D) + row;
#pragma unroll 1
      for (int d = 0; d < D; d += 32) {
        uint32_t o[32];
        tmem_ld32(tO + d, o);
        tmem_wait_ld(o);
        if (valid) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            dst[(d / 4 + k) * PROWS] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                                   __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
        }
      }
      tc_fence_before();
    }
  } else if (warp < LOAD_WARP + 4) {
    // ============================================================ loaders
    const int lw = warp - LOAD_WARP, lt = tid - LOAD_WARP * 32;
    int stage = 0;
    uint32_t eph = 1;
    bool alive = true;
    bool withhold = p.inject == 1;
    uint32_t raw_par = 0;  // parity of each raw slot's next completion
    fence_async_global();               // the copies below read what the ticket made visible
    uint32_t armed = 0, armed_par = 0;  // stages this warp has armed with copies, and the parity each was armed in
    // A tile's pages, one per lane (8 distinct), and whether a plain load of all
    // of them is right: every page in the pool, every token before the end.
    auto lookup = [&](int tile) -> int {
      const int pg = tile * PPAGES + (lane & 7);
      const int ph = pg < p.blocks ? __ldg(p.table + pg) : -1;
      return ph < p.num_pages ? ph : -1;
    };
    auto plain = [&](int tile, int ent) -> bool { return (tile + 1) * PTOK <= plen && __all_sync(0xffffffffu, ent >= 0); };
    auto advance = [&]() {
      if (++stage == ST) {
        stage = 0;
        eph ^= 1u;
      }
    };
    for (int g = g0; g < g1 && alive;) {
      PrefixSeg sg;
      g += prefix_segment(pl, g, g1, blockIdx.x, &sg);
      const int items = 2 * sg.tiles;
      bool is_v;
      int tile = sg.t0 + load_item(0, sg.tiles, sg.dual, &is_v);
      int ent = lookup(tile);
      // ---- K and V tiles
      if constexpr (!FP8) {
        for (int idx = 0; idx < items; ++idx) {
          const int t = tile, e = ent;
          const bool v = is_v;
          if (idx + 1 < items) {
            tile = sg.t0 + load_item(idx + 1, sg.tiles, sg.dual, &is_v);
            ent = lookup(tile);
          }
          if (!(alive = wait(&sh.empty[stage], eph))) break;
          const uint32_t full = smem_u32(&sh.full[stage]);
          const uint32_t dst = sKV + stage * C::TILE_BYTES;
          const bool all = plain(t, e);
          const int ph0 = __shfl_sync(0xffffffffu, e, 2 * lw), ph1 = __shfl_sync(0xffffffffu, e, 2 * lw + 1);
          if (withhold) {
            withhold = false;
          } else if (all) {
            if (lane == 0) {
              const CUtensorMap* map = v ? &p.tv : &p.tk;
              const uint32_t d0 = dst + 2 * lw * 2048;
              mbar_arrive_expect_tx(full, 2 * C::NH * 2048);
#pragma unroll
              for (int hf = 0; hf < C::NH; ++hf) {
                tma_load_5d(d0 + hf * HALF_BYTES, map, full, 0, 0, hf, sg.h, ph0);
                tma_load_5d(d0 + hf * HALF_BYTES + 2048, map, full, 0, 0, hf, sg.h, ph1);
              }
            }
            armed |= 1u << stage;
            armed_par = (armed_par & ~(1u << stage)) | ((eph ^ 1u) << stage);
          } else {
            // this warp's 32 rows, 16 bytes at a time
            constexpr int CPR = D / 8;
            const char* base = static_cast<const char*>(v ? p.v : p.k) + (v ? p.vp_h : p.kp_h) * 2 * sg.h;
            const long long sp = (v ? p.vp_p : p.kp_p) * 2, ss = (v ? p.vp_s : p.kp_s) * 2;
#pragma unroll 4
            for (int u = lane; u < 32 * CPR; u += 32) {
              const int r = u / CPR, ch = u % CPR, tok = t * PTOK + 32 * lw + r;
              const int ph = r < 16 ? ph0 : ph1;
              const bool ok = ph >= 0 && tok < plen;
              if (ph < 0 && tok < plen) sh.bad = 1;
              const int row = 32 * lw + r;
              cp_async16_zfill(dst + (ch >> 3) * HALF_BYTES + row * 128 + (((ch & 7) ^ (row & 7)) << 4),
                               ok ? base + ph * sp + (r & 15) * ss + ch * 16 : base, ok);
            }
            cp_async_commit();
            cp_async_wait<0>();
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(full);
          }
          advance();
        }
      } else {
        // e4m3: raw pages RAW - 1 tiles ahead; this warp widens its own 32 rows
        const uint32_t raw0 = sRaw + lw * 4096;
        // what is on the way: item, its pages, whether a TMA brings it
        int rt = tile;         // tile of the next request
        bool rv = is_v;
        int rent = ent;
        int req = 0;           // items requested
        int qt[RAW], qph0[RAW], qph1[RAW];
        bool qv[RAW], qall[RAW];
#pragma unroll
        for (int i = 0; i < RAW; ++i) qt[i] = qph0[i] = qph1[i] = 0, qv[i] = qall[i] = false;
        auto request = [&](int slot) {  // slot = req % RAW, a constant
          qt[slot] = rt;
          qv[slot] = rv;
          qall[slot] = plain(rt, rent);
          qph0[slot] = __shfl_sync(0xffffffffu, rent, 2 * lw);
          qph1[slot] = __shfl_sync(0xffffffffu, rent, 2 * lw + 1);
          if (qall[slot] && lane == 0) {
            const CUtensorMap* map = rv ? &p.tv : &p.tk;
            const uint32_t bar = smem_u32(&sh.raw[lw][slot]);
            mbar_arrive_expect_tx(bar, 4096);
            tma_load_4d(raw0 + slot * HALF_BYTES, map, bar, 0, 0, sg.h, qph0[slot]);
            tma_load_4d(raw0 + slot * HALF_BYTES + 2048, map, bar, 0, 0, sg.h, qph1[slot]);
          }
          if (++req < items) {
            rt = sg.t0 + load_item(req, sg.tiles, sg.dual, &rv);
            rent = lookup(rt);
          }
        };
#pragma unroll
        for (int i = 0; i < RAW - 1; ++i)
          if (req < items) request(i);
        for (int i0 = 0; i0 < items && alive; i0 += RAW) {
#pragma unroll
          for (int sl = 0; sl < RAW; ++sl) {
            const int idx = i0 + sl;
            if (idx >= items) break;
            // the slot that the previous item left is requested anew
            if (req < items) request((sl + RAW - 1) % RAW);
            const int t = qt[sl], ph0 = qph0[sl], ph1 = qph1[sl];
            // lane: rows (lane >> 3) + 4 k, 16-byte chunk lane & 7 (16 elements)
            const int ch = lane & 7, r0 = lane >> 3;
            uint4 x[8];
            if (qall[sl]) {
              if (!(alive = wait(&sh.raw[lw][sl], (raw_par >> sl) & 1u))) break;
              raw_par ^= 1u << sl;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int r = r0 + 4 * k;
                x[k] = lds128(raw0 + sl * HALF_BYTES + r * 128 + ((ch ^ (r & 7)) << 4));
              }
            } else {
              const unsigned char* base = static_cast<const unsigned char*>(qv[sl] ? p.v : p.k) + (qv[sl] ? p.vp_h : p.kp_h) * sg.h;
              const long long sp = qv[sl] ? p.vp_p : p.kp_p, ss = qv[sl] ? p.vp_s : p.kp_s;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int r = r0 + 4 * k, tok = t * PTOK + 32 * lw + r;
                const int ph = r < 16 ? ph0 : ph1;
                if (ph < 0 && tok < plen) sh.bad = 1;
                x[k] = make_uint4(0u, 0u, 0u, 0u);
                if (ph >= 0 && tok < plen) x[k] = __ldg(reinterpret_cast<const uint4*>(base + ph * sp + (r & 15) * ss + ch * 16));
              }
            }
            if (!(alive = wait(&sh.empty[stage], eph))) break;
            const uint32_t dst = sKV + stage * C::TILE_BYTES + (ch >> 2) * HALF_BYTES + 32 * lw * 128;
            const int c0 = (2 * ch) & 7;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int r = r0 + 4 * k;
              uint32_t w[8];
              e4m3x4_to_f16x2x2(x[k].x, w[0], w[1]);
              e4m3x4_to_f16x2x2(x[k].y, w[2], w[3]);
              e4m3x4_to_f16x2x2(x[k].z, w[4], w[5]);
              e4m3x4_to_f16x2x2(x[k].w, w[6], w[7]);
              // lanes of the upper half store their second chunk first: a row's
              // eight lanes then fill eight different 16-byte columns at a time
              const uint32_t d0 = dst + r * 128 + ((c0 ^ (r & 7)) << 4), d1 = dst + r * 128 + (((c0 + 1) ^ (r & 7)) << 4);
              const bool up = ch >= 4;
              sts128(up ? d1 : d0, up ? w[4] : w[0], up ? w[5] : w[1], up ? w[6] : w[2], up ? w[7] : w[3]);
              sts128(up ? d0 : d1, up ? w[0] : w[4], up ? w[1] : w[5], up ? w[2] : w[6], up ? w[3] : w[7]);
            }
            // also orders the reads of the raw slot before its next copy
            fence_async_proxy();
            __syncwarp();
            if (lane == 0 && !withhold) mbar_arrive(smem_u32(&sh.full[stage]));
            withhold = false;
            advance();
          }
        }
      }
    }
    // A wait ran out: let the copies in flight land before the block exits.
    cp_async_wait<0>();
    if (!alive && lane == 0) {
      if constexpr (FP8) {
        for (int i = 0; i < RAW; ++i) mbar_wait(smem_u32(&sh.raw[lw][i]), (raw_par >> i) & 1u, p.wait_ns);
      } else {
        for (int i = 0; i < ST; ++i)
          if ((armed >> i) & 1u) mbar_wait(smem_u32(&sh.full[i]), (armed_par >> i) & 1u, p.wait_ns);
      }
    }
    if (sh.bad && lane == 0 && p.status != nullptr) atomicOr(p.status, FK_STATUS_BAD_PAGE);
  } else {
    // ============================================================ MMA issue (the whole warp walks, one lane issues)
    constexpr uint32_t idQK = instr_desc(MBF16, PROWS, PITEM, false);
    constexpr uint32_t idPV = instr_desc(MBF16, PROWS, D, true);
    int stage = 0;
    uint32_t fph = 0, qph = 0, pph[2] = {0, 0};  // pph[s]: parities of the stream's two P buffers
    bool alive = true;
    const bool leader = elect_one();
    // S = Q K^T of stream s, item buffer buf: Q of row tile qt, 64 rows of K at k_addr
    auto qk = [&](int s, int buf, int qt, uint32_t k_addr) {
      const uint32_t q_lo = desc_lo(sQ + qt * C::TILE_BYTES, 16), k_lo = desc_lo(k_addr, 16);
      if (leader) {
        mma_ss<false>(s * 128 + buf * PITEM, q_lo, k_lo, idQK);
#pragma unroll
        for (int k = 1; k < D / 16; ++k) {
          const uint32_t off = ((k >> 2) * HALF_BYTES + (k & 3) * 32) >> 4;
          mma_ss<true>(s * 128 + buf * PITEM, q_lo + off, k_lo + off, idQK);
        }
        mma_commit(smem_u32(&sh.s[s][buf]));
      }
    };
    // O (+)= P V of stream s, item buffer buf: 64 rows of V at v_addr
    auto pv = [&](int s, int buf, uint32_t v_addr, int j, int ni) {
      const uint32_t v_lo = desc_lo(v_addr, HALF_BYTES);
      if (leader) {
#pragma unroll
        for (int k = 0; k < PITEM / 16; ++k)
          mma_ts(256 + s * D, s * 128 + buf * PITEM + 8 * k, v_lo + k * (2048 >> 4), idPV, j > 0 || k > 0);
        if (j + 2 == ni) mma_commit(smem_u32(&sh.o[s]));
        if (j + 1 == ni) mma_commit(smem_u32(&sh.done[s]));
      }
    };
    for (int g = g0; g < g1 && alive;) {
      PrefixSeg sg;
      g += prefix_segment(pl, g, g1, blockIdx.x, &sg);
      const bool dual = sg.dual;
      const int ni = dual ? 2 * sg.tiles : sg.tiles;
      // Item j of stream s: dual, 64-token half j & 1 of token tile j / 2;
      // parity, half s of token tile j.
      auto half_of = [&](int s, int j) -> uint32_t { return (dual ? (j & 1) : s) * (PITEM * 128); };
      if (!(alive = wait(&sh.qfull, qph))) break;
      qph ^= 1u;
      auto give_back = [&](int st) {
        if (leader) mma_commit(smem_u32(&sh.empty[st]));
      };
      auto advance = [&]() {
        if (++stage == ST) {
          stage = 0;
          fph ^= 1u;
        }
      };
      // two items of S ahead of the softmax
      for (int j = 0; j < min(ni, 2) && alive; ++j) {
        if (!dual || j == 0) alive = wait(&sh.full[stage], fph);
        if (!alive) break;
        const uint32_t k_addr = sKV + stage * C::TILE_BYTES;
        qk(0, j, 0, k_addr + half_of(0, j));
        qk(1, j, dual ? 1 : 0, k_addr + half_of(1, j));
        if (!dual || j == 1) {
          give_back(stage);
          advance();
        }
      }
      // step j: P V of item j, S of item j + 2; the ring holds V at its head and
      // K behind it (for two steps with dual)
      for (int j = 0; j < ni && alive; ++j) {
        const int buf = j & 1;
        const bool first_use = !dual || buf == 0, last_use = !dual || buf == 1, more = j + 2 < ni;
        if (first_use && !(alive = wait(&sh.full[stage], fph))) break;
        const int ks = stage + 1 == ST ? 0 : stage + 1;
        const uint32_t kph = stage + 1 == ST ? fph ^ 1u : fph;
        const uint32_t v_addr = sKV + stage * C::TILE_BYTES, k_addr = sKV + ks * C::TILE_BYTES;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (!(alive = wait(&sh.p[s][buf], (pph[s] >> buf) & 1u))) break;
          pph[s] ^= 1u << buf;
          tc_fence_after();
          pv(s, buf, v_addr + half_of(s, j), j, ni);
          if (s == 1 && last_use) give_back(stage);
          if (more) {
            if (s == 0 && first_use && !(alive = wait(&sh.full[ks], kph))) break;
            qk(s, buf, dual ? s : 0, k_addr + half_of(s, j));
            if (s == 1 && last_use) give_back(ks);
          }
        }
        if (!alive) break;
        if (last_use) {
          advance();
          if (more) advance();
        }
      }
      if (!alive) break;
      if (leader) mma_commit(smem_u32(&sh.qempty));
    }
    // nothing of this warp's is in flight when the tensor memory is given back
    if (leader) mma_commit(smem_u32(&sh.drain));
    mbar_wait(smem_u32(&sh.drain), 0, p.wait_ns);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_wait();
  if (warp == MMA_WARP) tmem_dealloc(*const_cast<volatile uint32_t*>(&sh.tmem), 512);
}

// ------------------------------------------------------------------------
// Join: out = (sum_i 2^(m_i - M) acc_i) / (sum_i 2^(m_i - M) l_i [+ 2^(s - M)])
// over the prefix segments of the row and its own part, in one pass with a
// running maximum.  A thread has one row and four dims and keeps eight records'
// loads in flight; a warp reads 512 contiguous bytes of a record.  With fewer
// rows than threads the block takes more dims instead.
// ------------------------------------------------------------------------
struct JoinParams {
  const float2* ml;       // prefix segments
  const float* acc;
  OwnRecords own;
  const int* plan;        // granules of a prefix CTA
  unsigned long long* ticket;
  const int* plen_dev;
  int plen, blocks, rows, G, kv_heads;
  const float* s_aux;
  const float* scale_v;
  void* out;
  long long o_b, o_h;
  int out_dtype, o_al8;
  int rb;  // rows of a block (a power of two); JTHREADS / rb groups of four dims
};

constexpr int JTHREADS = 128;
constexpr int JBATCH = 8;  // prefix records of a row in flight
constexpr int JOWN = 4;    // own records

template <int D>
__global__ void __launch_bounds__(JTHREADS) join_kernel(const __grid_constant__ JoinParams p) {
  grid_dependency_wait();
  grid_dependency_trigger();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.ticket = 0;  // a graph replays its ticket
  const int per = __ldcg(p.plan);
  const int per_head = (p.rows + p.rb - 1) / p.rb;
  const int h = blockIdx.x / per_head, first = blockIdx.x % per_head * p.rb;  // the block's first row
  const int tile = first / PROWS, row = first % PROWS + (threadIdx.x & (p.rb - 1));
  const int grow = tile * PROWS + row;
  const int d0 = (blockIdx.y * (JTHREADS / p.rb) + threadIdx.x / p.rb) * 4;
  if (grow >= p.rows || d0 >= D) return;
  const int b = grow / p.G, qh = h * p.G + grow % p.G;
  int item, slot;
  p.own.find(h, grow % p.G, &item, &slot);
  const long long oitem = static_cast<long long>(b) * p.own.per_seq + item;
  const int2 own = p.own.of(oitem);  // needed last: the prefix's records are read meanwhile
  bool past;
  const int plen = prefix_len(p.plen_dev, p.plen, p.blocks, &past);
  const PrefixPlan pl(plen, p.rows, p.kv_heads);
  const int unit = tile >> 1;
  const bool dual = unit < pl.nd;
  long long rec0 = 0;  // the row's records: every (dual) second one from rec0 on
  int nrec = 0;
  if (pl.nt > 0) {
    const int base = h * pl.gh + pl.unit_base(unit);
    const int c0 = base / per, c1 = (base + pl.unit_len(unit) - 1) / per;
    rec0 = 2ll * (c0 + h * pl.upu + unit) + (dual ? (tile & 1) : 0);
    nrec = (c1 - c0 + 1) * (dual ? 1 : 2);
  }
  const int rstep = dual ? 2 : 1;

  float M = NEG_INF, L = 0.f;
  float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
  auto merge = [&](const auto& ml, const auto& av, auto count) {
    constexpr int N = decltype(count)::value;
    float Mn = M;
#pragma unroll
    for (int k = 0; k < N; ++k) Mn = max3_nan(Mn, ml[k].x, ml[k].x);
    if (Mn == NEG_INF) return;
    const float sc = exp2f(M - Mn);
    L *= sc;
    A.x *= sc;
    A.y *= sc;
    A.z *= sc;
    A.w *= sc;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (ml[k].x == NEG_INF) continue;  // nothing attended: the accumulators may be unwritten
      const float e = exp2f(ml[k].x - Mn);
      L += e * ml[k].y;
      A.x += e * av[k].x;
      A.y += e * av[k].y;
      A.z += e * av[k].z;
      A.w += e * av[k].w;
    }
    M = Mn;
  };
  const float2 none = make_float2(NEG_INF, 0.f);
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < nrec; i += JBATCH) {
    float2 ml[JBATCH];
    float4 av[JBATCH];
#pragma unroll
    for (int k = 0; k < JBATCH; ++k) {
      const bool ok = i + k < nrec;
      const long long rec = rec0 + static_cast<long long>(i + k) * rstep;
      ml[k] = ok ? __ldcg(p.ml + rec * PROWS + row) : none;
      av[k] = ok ? __ldcg(reinterpret_cast<const float4*>(p.acc + rec * PROWS * D) + (d0 / 4) * PROWS + row) : zero;
    }
    merge(ml, av, std::integral_constant<int, JBATCH>{});
  }
  for (int i = 0; i < own.y; i += JOWN) {
    float2 ml[JOWN];
    float4 av[JOWN];
#pragma unroll
    for (int k = 0; k < JOWN; ++k) {
      const bool ok = i + k < own.y;
      const long long rec = (oitem + own.x + i + k) * p.own.slots + slot;
      ml[k] = ok ? __ldcg(p.own.ml + rec) : none;
      if (ml[k].y != ml[k].y) ml[k].x = ml[k].y;  // the own part's maximum passes NaN by, its sum does not
      av[k] = ok ? __ldcg(reinterpret_cast<const float4*>(p.own.acc + rec * HEAD_DIM + d0)) : zero;
    }
    merge(ml, av, std::integral_constant<int, JOWN>{});
  }
  float e, Lf;
  if (M == NEG_INF) e = 0.f, Lf = 0.f;  // nothing attended: zeros, whatever the sink
  else sink_norm(L, M, p.s_aux, qh, &e, &Lf);
  const float sv = p.scale_v != nullptr ? __ldg(p.scale_v) : 1.f;
  const float f = Lf == 0.f ? 0.f : sv;  // a NaN stays one
  const float o0 = f == 0.f ? 0.f : A.x * e / Lf * f, o1 = f == 0.f ? 0.f : A.y * e / Lf * f,
              o2 = f == 0.f ? 0.f : A.z * e / Lf * f, o3 = f == 0.f ? 0.f : A.w * e / Lf * f;
  const long long ob = b * p.o_b + qh * p.o_h + d0;
  const bool bf = p.out_dtype == FK_DTYPE_BF16;
  if (p.o_al8) {
    *reinterpret_cast<uint2*>(static_cast<unsigned short*>(p.out) + ob) =
        bf ? make_uint2(pack2<true>(o0, o1), pack2<true>(o2, o3)) : make_uint2(pack2<false>(o0, o1), pack2<false>(o2, o3));
  } else {
    const float o[4] = {o0, o1, o2, o3};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (bf) static_cast<__nv_bfloat16*>(p.out)[ob + i] = __float2bfloat16_rn(o[i]);
      else static_cast<__half*>(p.out)[ob + i] = __float2half_rn(o[i]);
    }
  }
}

// ------------------------------------------------------------------------
// Host side.
// ------------------------------------------------------------------------
namespace {

int prefix_ctas(int device) {
  int sms = 0;
  return cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) == cudaSuccess ? sms : 0;
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// A word that no scratch holds by accident or from an earlier call: the time of
// the first call, its bits spread over the word, counted up.  Odd: never 0.
unsigned long long next_ticket() {
  static std::atomic<unsigned long long> next{
      static_cast<unsigned long long>(std::chrono::steady_clock::now().time_since_epoch().count()) * 0x9e3779b97f4a7c15ull | 1ull};
  return next.fetch_add(2);
}

// [own part's decode workspace | its items' records | plan, ticket | prefix (max, sum) | prefix acc]
struct PrefixWs {
  size_t own, info, plan, ml, acc, total;
  PrefixWs(int device, int batch, int q_heads, int kv_heads, int head_dim, int kv_dtype) {
    own = fk_decode_workspace_bytes_gqa(device, batch, q_heads, kv_heads, kv_dtype);
    const long long rows = static_cast<long long>(batch) * (q_heads / kv_heads);
    const size_t rt = static_cast<size_t>((rows + PROWS - 1) / PROWS);
    const size_t segs = static_cast<size_t>(prefix_ctas(device)) + static_cast<size_t>(kv_heads) * ((rt + 1) / 2);
    const size_t items = static_cast<size_t>(batch) * q_heads;  // at most
    info = up256(own);
    plan = up256(info + items * sizeof(int2));
    ml = plan + 256;
    acc = up256(ml + segs * 2 * PROWS * sizeof(float2));
    total = own == 0 ? 0 : up256(acc + segs * 2 * PROWS * head_dim * sizeof(float));
  }
};

template <int KV, int D>
int launch_prefix(const PrefixParams& p, int ctas, int device, cudaStream_t stream) {
  static bool done[64] = {};
  static std::mutex mu;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!done[device]) {
      const cudaError_t e = cudaFuncSetAttribute(prefix_kernel<KV, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, prefix_smem<KV, D>());
      if (e != cudaSuccess) return fail(FK_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      done[device] = true;
    }
  }
  const cudaError_t e = launch_pdl(prefix_kernel<KV, D>, dim3(ctas), dim3(PTHREADS), prefix_smem<KV, D>(), stream, p);
  return e == cudaSuccess ? FK_OK : fail(FK_ERR_CUDA, "prefix launch failed: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace fk

using namespace fk;

extern "C" size_t fk_shared_prefix_workspace_bytes(int device, int batch, int q_heads, int kv_heads, int head_dim,
                                                   int kv_dtype) {
  if (batch < 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0 || (head_dim != 64 && head_dim != 128)) {
    fail(FK_ERR_INVALID_ARG, "bad sizes");
    return 0;
  }
  return PrefixWs(device, batch, q_heads, kv_heads, head_dim, kv_dtype).total;
}

extern "C" int fk_paged_shared_prefix_decode(const fk_prefix_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (a == nullptr) return fail(FK_ERR_INVALID_ARG, "args must be non-null");
  if (a->batch == 0) return FK_OK;
  if (a->batch < 0 || a->q_heads <= 0 || a->kv_heads <= 0 || a->batch > 0x7fffffffLL || a->q_heads > 65535 ||
      a->kv_heads > 65535 || a->batch * a->q_heads > 0x7fffffffLL)
    return fail(FK_ERR_INVALID_ARG, "bad sizes: batch=%lld q_heads=%lld kv_heads=%lld", static_cast<long long>(a->batch),
                static_cast<long long>(a->q_heads), static_cast<long long>(a->kv_heads));
  if (a->num_pages <= 0 || a->num_pages > 0x7fffffffLL || a->max_blocks < 0 || a->max_blocks > 0x7fffffffLL ||
      a->prefix_blocks < 0 || a->prefix_blocks > 0x7ffffffLL || a->prefix_len < 0 || a->prefix_len > 0x7fffff00LL)
    return fail(FK_ERR_INVALID_ARG, "bad page counts or prefix length");
  {
    // granules of the prefix part (see PrefixPlan), and the CTAs added to them
    const long long rt = (a->batch * (a->q_heads / a->kv_heads) + PROWS - 1) / PROWS, nt = (a->prefix_blocks * PAGE + PTOK - 1) / PTOK;
    if (a->q_heads % a->kv_heads == 0 && a->kv_heads * ((rt + 1) / 2) * nt > (1ll << 30))
      return fail(FK_ERR_UNSUPPORTED, "too many row tiles x prefix pages (%lld x %lld)", static_cast<long long>(a->kv_heads * rt),
                  static_cast<long long>(a->prefix_blocks));
  }
  if (a->prefix_table == nullptr && a->prefix_blocks > 0) return fail(FK_ERR_INVALID_ARG, "prefix_table must be non-null");
  OwnPart own;
  int device = 0;
  int rc = own_part_prepare(&own, *a, workspace, &device);
  if (rc != FK_OK) return rc;
  const int B = static_cast<int>(a->batch), QH = static_cast<int>(a->q_heads), KVH = static_cast<int>(a->kv_heads);
  const int D = static_cast<int>(a->head_dim), kv = static_cast<int>(a->kv_dtype);
  const PrefixWs w(device, B, QH, KVH, D, kv);
  if (w.total == 0) return FK_ERR_CUDA;
  if (workspace_bytes < w.total)
    return fail(FK_ERR_WORKSPACE, "workspace too small: %zu bytes < %zu required", workspace_bytes, w.total);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const int ctas = prefix_ctas(device);
  PrefixParams p = {};
  p.q = a->q;
  p.q_b = a->q_b;
  p.q_h = a->q_h;
  p.k = a->k_pool;
  p.v = a->v_pool;
  p.kp_p = a->kp_p;
  p.kp_h = a->kp_h;
  p.kp_s = a->kp_s;
  p.vp_p = a->vp_p;
  p.vp_h = a->vp_h;
  p.vp_s = a->vp_s;
  p.table = static_cast<const int*>(a->prefix_table);
  p.plen_dev = static_cast<const int*>(a->prefix_len_dev);
  p.plen = static_cast<int>(a->prefix_len);
  p.blocks = static_cast<int>(a->prefix_blocks);
  p.num_pages = static_cast<int>(a->num_pages);
  p.G = QH / KVH;
  p.rows = B * p.G;
  p.kv_heads = KVH;
  p.q_dtype = static_cast<int>(a->q_dtype);
  p.q_al16 = own.q_al16;
  p.scale_q = p.q_dtype == FK_DTYPE_E4M3 ? static_cast<const float*>(a->scale_q) : nullptr;
  p.scale_k = kv == FK_DTYPE_E4M3 ? static_cast<const float*>(a->scale_k) : nullptr;
  p.ml = reinterpret_cast<float2*>(ws + w.ml);
  p.acc = reinterpret_cast<float*>(ws + w.acc);
  p.status = static_cast<int*>(a->status);
  debug_settings(&p.wait_ns, &p.inject);
  // 16-bit: (64 dims, 16 slots, D / 64 halves, heads, pages), a box is one
  // half of a page; e4m3: (128 dims, 16 slots, heads, pages), a box is a page
  for (int i = 0; i < 2; ++i) {
    const void* base = i == 0 ? p.k : p.v;
    const uint64_t sp = static_cast<uint64_t>(i == 0 ? p.kp_p : p.vp_p), sh = static_cast<uint64_t>(i == 0 ? p.kp_h : p.vp_h),
                   ss = static_cast<uint64_t>(i == 0 ? p.kp_s : p.vp_s);
    if (kv == FK_DTYPE_E4M3) {
      const uint64_t dims[4] = {128, PAGE, static_cast<uint64_t>(KVH), static_cast<uint64_t>(a->num_pages)};
      const uint64_t strides[3] = {ss, sh, sp};
      const uint32_t box[4] = {128, PAGE, 1, 1};
      rc = encode_map(i == 0 ? &p.tk : &p.tv, kv, 4, base, dims, strides, box);
    } else {
      const uint64_t dims[5] = {64, PAGE, static_cast<uint64_t>(D / 64), static_cast<uint64_t>(KVH), static_cast<uint64_t>(a->num_pages)};
      const uint64_t strides[4] = {2 * ss, 128, 2 * sh, 2 * sp};
      const uint32_t box[5] = {64, PAGE, 1, 1, 1};
      rc = encode_map(i == 0 ? &p.tk : &p.tv, kv, 5, base, dims, strides, box);
    }
    if (rc != FK_OK) return rc;
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  DeviceScope scope(device);
  JoinParams j = {};
  p.ticket = j.ticket = reinterpret_cast<unsigned long long*>(ws + w.plan + 128);
  p.ticket_value = next_ticket();
  rc = own_part_launch(own, reinterpret_cast<int2*>(ws + w.info), j.ticket, p.ticket_value, p.status, w.own, st, &j.own);
  if (rc != FK_OK) return rc;
  p.seq_lens = static_cast<const int*>(a->seq_lens);
  p.batch = B;
  p.own_items = j.own.per_seq;
  j.plan = p.plan = reinterpret_cast<int*>(ws + w.plan);
  if (kv == FK_DTYPE_F16) rc = D == 64 ? launch_prefix<FK_DTYPE_F16, 64>(p, ctas, device, st) : launch_prefix<FK_DTYPE_F16, 128>(p, ctas, device, st);
  else if (kv == FK_DTYPE_BF16) rc = D == 64 ? launch_prefix<FK_DTYPE_BF16, 64>(p, ctas, device, st) : launch_prefix<FK_DTYPE_BF16, 128>(p, ctas, device, st);
  else rc = launch_prefix<FK_DTYPE_E4M3, 128>(p, ctas, device, st);
  if (rc != FK_OK) return rc;
  j.ml = p.ml;
  j.acc = p.acc;
  j.plen_dev = p.plen_dev;
  j.plen = p.plen;
  j.blocks = p.blocks;
  j.rows = p.rows;
  j.G = p.G;
  j.kv_heads = KVH;
  j.s_aux = static_cast<const float*>(a->s_aux);
  j.scale_v = kv == FK_DTYPE_E4M3 ? static_cast<const float*>(a->scale_v) : nullptr;
  j.out = a->out;
  j.o_b = a->o_b;
  j.o_h = a->o_h;
  j.out_dtype = static_cast<int>(a->out_dtype);
  j.o_al8 = own.p.o_al8;
  j.rb = 8;
  while (j.rb < PROWS && j.rb < p.rows) j.rb *= 2;
  const dim3 grid(static_cast<unsigned>(KVH * ((p.rows + j.rb - 1) / j.rb)), static_cast<unsigned>((D / 4 * j.rb + JTHREADS - 1) / JTHREADS));
  const cudaError_t e = D == 128 ? launch_pdl(join_kernel<128>, grid, dim3(JTHREADS), 0, st, j)
                                 : launch_pdl(join_kernel<64>, grid, dim3(JTHREADS), 0, st, j);
  return e == cudaSuccess ? FK_OK : fail(FK_ERR_CUDA, "join launch failed: %s", cudaGetErrorString(e));
}
