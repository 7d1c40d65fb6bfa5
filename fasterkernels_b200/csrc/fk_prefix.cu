// fk_prefix.cu -- decode attention of a batch whose sequences share a prefix.
//
// Sequence b attends the prefix's P tokens and then its own.  Softmax
// statistics join by log-sum-exp, so the two parts are computed apart: the
// prefix once for the whole batch (below), the own tokens by the split-KV
// decode kernel (fk_decode_kernel.cuh), which stores its running (max, sum,
// acc) instead of an output; a last kernel joins them with the sink.
//
// Prefix part.  For one KV head the batch's query heads are the rows of a
// matrix: row r = b * G + g, R = B * G rows, and the work is S = Q K^T (R x P),
// a softmax numerator per row and O = P V.  Reading the prefix once for up to
// 256 rows turns a read of B x P tokens into a matrix product of 4 R P D
// operations per KV head on 2 P D elements: tensor cores, not memory, carry it
// from about 256 rows on.
//
//   tcgen05 tiles of 128 rows x 128 tokens; S (f32, 128 columns) and O (f32, D
//   columns) live in tensor memory, two of each, so that two independent
//   streams alternate: while one stream's softmax runs on the CUDA cores, the
//   tensor cores work for the other.  With more than 128 rows the streams are
//   two row tiles that share each K / V tile (dual); otherwise they are the
//   even and the odd token tiles of one row tile (parity).
//   P (f16, or bf16 for bf16 KV) overwrites the first half of its own S in
//   tensor memory and is the A operand of O += P V from there.
//
// Work is cut like the decode kernel's: units (KV head, one or two row tiles)
// laid end to end in granules (dual: one token tile, parity: two), each CTA of
// the persistent grid takes an equal run of them, and the piece of a unit in a
// CTA is a segment whose (max, sum, O) goes to the workspace.  Planned on the
// device from the prefix length.
//
// Warps: 0-3 and 4-7 softmax of stream 0 and 1 (thread = row), 8-11 load Q, K
// and V, 12 issues the MMAs.  Loads are cp.async (16-bit) or loads widened to
// f16 in registers (e4m3) rather than TMA: pages are 16 tokens, and a K or V
// tile that the tensor cores read with one descriptor needs its 8-row groups
// evenly spaced, which a page-sized box of two 128-byte halves does not leave;
// cp.async also writes zeros for tokens past the prefix and for bad pages.
#include <cuda_fp8.h>

#include "fk_decode_kernel.cuh"
#include "fk_host.h"
#include "fk_prefix.h"
#include "fk_tc.cuh"

namespace fk {

constexpr int PROWS = 128;    // rows of a row tile (MMA M)
constexpr int PTOK = 128;     // tokens of a token tile (MMA N of QK, K of PV)
constexpr int PPAGES = PTOK / PAGE;
constexpr int PTHREADS = 13 * 32;
constexpr int HALF_BYTES = PTOK * 128;  // 128 rows of a 128-byte half
constexpr int LOAD_LAG = 2;   // K / V tiles a loader issues ahead of the one it publishes

template <int D>
struct PCfg {
  static constexpr int NH = D / 64;
  static constexpr int TILE_BYTES = NH * HALF_BYTES;  // Q, K or V tile in 16 bits
  static constexpr int STAGES = D == 128 ? 5 : 8;
  static constexpr int SMEM = 1024 + (2 + STAGES) * TILE_BYTES + 512;
};

struct PrefixParams {
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
  float2* ml;
  float* acc;
  int* zero;            // the own part's status word and arrival counters
  int zero_words;
  int* status;          // or null
  unsigned long long wait_ns;
  int inject;
};

// Granules and units, from the prefix length (device side).
struct PrefixPlan {
  int nt, nd, upu;       // token tiles; dual units and units of a KV head
  long long gh, total, per;
  __device__ PrefixPlan(int plen, int rows, int kv_heads, int ctas) {
    const int rt = (rows + PROWS - 1) / PROWS;
    nt = (plen + PTOK - 1) / PTOK;
    nd = rt / 2;
    upu = nd + (rt & 1);
    gh = static_cast<long long>(nd) * nt + ((rt & 1) ? (nt + 1) / 2 : 0);
    total = gh * kv_heads;
    per = max((total + ctas - 1) / ctas, 1ll);
  }
  // First granule and length of unit u of a KV head.
  __device__ long long unit_base(int u) const { return static_cast<long long>(u) * nt; }
  __device__ int unit_len(int u) const { return u < nd ? nt : (nt + 1) / 2; }
};

struct PrefixSeg {
  int h, unit, seg, dual, t0, tiles;  // token tiles [t0, t0 + tiles)
};

// The segment at granule g of CTA c (granules [.., end)); returns its length.
__device__ __forceinline__ long long prefix_segment(const PrefixPlan& pl, long long g, long long end, int c, PrefixSeg* s) {
  s->h = static_cast<int>(g / pl.gh);
  const long long r = g - s->h * pl.gh;
  const long long dualg = static_cast<long long>(pl.nd) * pl.nt;
  s->dual = r < dualg;
  s->unit = s->dual ? static_cast<int>(r / pl.nt) : pl.nd;
  const int off = static_cast<int>(r - pl.unit_base(s->unit));
  const long long n = min(end - g, static_cast<long long>(pl.unit_len(s->unit) - off));
  s->seg = c + s->h * pl.upu + s->unit;
  s->t0 = s->dual ? off : 2 * off;
  s->tiles = s->dual ? static_cast<int>(n) : static_cast<int>(min(2 * n, static_cast<long long>(pl.nt - 2 * off)));
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
  using C = PCfg<D>;
  constexpr bool FP8 = KV == FK_DTYPE_E4M3;
  constexpr bool MBF16 = KV == FK_DTYPE_BF16;
  constexpr int ST = C::STAGES;
  // f16 P is stored times 2^BIAS: with at most 2^8 above the reference maximum
  // it stays below 2^15, and the smallest P that does not vanish is 2^-32 of the
  // maximum's instead of 2^-25 (bf16 has f32's range and needs none).
  constexpr float BIAS = MBF16 ? 0.f : 7.f;
  constexpr float LAZY = 8.f;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = smem;                           // [2] row tiles
  const uint32_t sKV = smem + 2 * C::TILE_BYTES;      // [ST]
  __shared__ __align__(8) uint64_t b_full[ST], b_empty[ST], b_qfull, b_qempty, b_s[2], b_p[2], b_o[2], b_drain;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_bad;  // a bad page was seen: the softmax checks pages from then on
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(smem_u32(&b_full[i]), 4);
      mbar_init(smem_u32(&b_empty[i]), 1);
    }
    mbar_init(smem_u32(&b_qfull), 4);
    mbar_init(smem_u32(&b_qempty), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&b_s[i]), 1);
      mbar_init(smem_u32(&b_p[i]), 4);
      mbar_init(smem_u32(&b_o[i]), 1);
    }
    mbar_init(smem_u32(&b_drain), 1);
    fence_mbar_init();
    s_bad = 0;
  }
  if (warp == 12) tmem_alloc(smem_u32(&s_tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *const_cast<volatile uint32_t*>(&s_tmem);
  grid_dependency_wait();
  grid_dependency_trigger();
  for (int i = blockIdx.x * PTHREADS + tid; i < p.zero_words; i += gridDim.x * PTHREADS) p.zero[i] = 0;

  const int plen = max(p.plen_dev != nullptr ? __ldg(p.plen_dev) : p.plen, 0);
  const PrefixPlan pl(plen, p.rows, p.kv_heads, gridDim.x);
  const long long g0 = blockIdx.x * pl.per, g1 = min(g0 + pl.per, pl.total);
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

  if (warp < 8) {
    // ============================================================ softmax
    const int s = warp >> 2;
    const int row = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // lane (warp & 3) * 32 in bits 16..
    const uint32_t tS = tmem + lanes + s * 128, tO = tmem + lanes + 256 + s * D;
    // never 0: a masked logit (-inf) stays one
    const float c = fmaxf(rsqrtf(static_cast<float>(D)) * LOG2E * fabsf(sk), 1e-30f);
    uint32_t sph = 0, oph = 0;
    bool alive = true;
    for (long long g = g0; g < g1 && alive;) {
      PrefixSeg sg;
      g += prefix_segment(pl, g, g1, blockIdx.x, &sg);
      const int n = sg.dual ? sg.tiles : (sg.tiles + 1 - s) / 2;  // token tiles of this stream
      const int trow = (2 * sg.unit + (sg.dual ? s : 0)) * PROWS + row;
      float m = NEG_INF, l = 0.f;
      for (int i = 0; i < n; ++i) {
        const int tile = sg.t0 + (sg.dual ? i : 2 * i + s);
        if (!(alive = wait(&b_s[s], sph))) break;
        sph ^= 1u;
        tc_fence_after();
        const int lim = plen - tile * PTOK;  // tokens of the tile that exist
        uint32_t okp = 0xffu;                // its pages that do
        if (s_bad) {
          okp = 0;
          for (int j = 0; j < PPAGES; ++j) {
            const int pg = tile * PPAGES + j;
            const int ph = pg < p.blocks ? __ldg(p.table + pg) : -1;
            okp |= (ph >= 0 && ph < p.num_pages ? 1u : 0u) << j;
          }
        }
        const bool masked = lim < PTOK || okp != 0xffu;
        auto mask = [&](uint32_t (&r)[32], int col) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (col + j >= lim || !((okp >> ((col + j) >> 4)) & 1u)) r[j] = __float_as_uint(NEG_INF);
        };
        // ---- the row's maximum
        uint32_t ra[32], rb[32];
        float mx0 = NEG_INF, mx1 = NEG_INF, mx2 = NEG_INF, mx3 = NEG_INF;
        auto maxes = [&](uint32_t (&r)[32]) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            mx0 = fmaxf(mx0, __uint_as_float(r[j]));
            mx1 = fmaxf(mx1, __uint_as_float(r[j + 1]));
            mx2 = fmaxf(mx2, __uint_as_float(r[j + 2]));
            mx3 = fmaxf(mx3, __uint_as_float(r[j + 3]));
          }
        };
        tmem_ld32(tS, ra);
#pragma unroll
        for (int ch = 0; ch < 4; ch += 2) {
          tmem_wait_ld(ra);
          tmem_ld32(tS + 32 * (ch + 1), rb);
          if (masked) mask(ra, 32 * ch);
          maxes(ra);
          tmem_wait_ld(rb);
          if (ch == 0) tmem_ld32(tS + 64, ra);
          if (masked) mask(rb, 32 * ch + 32);
          maxes(rb);
        }
        const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * c;
        // The reference maximum moves only when a logit exceeds it by more than
        // LAZY (log2 units): any reference gives the same softmax once O and l
        // are normalised together, and O is rescaled in the first tiles only.
        const bool grow = mx > m + LAZY;
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = grow ? mx : m;
          const float al = (m == NEG_INF) ? 0.f : ex2(m - mn);
          l *= al;
          if (i > 0) {
            // S of this tile is complete, hence so is every earlier P V of this stream
            uint32_t o[32];
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
              tmem_ld32(tO + d, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * al);
              tmem_st32(tO + d, o);
            }
          }
          m = mn;
        }
        const float mb = (m == NEG_INF ? 0.f : m) - BIAS;
        // ---- P = 2^(x - m + BIAS), 32 columns at a time
        tmem_ld32(tS, ra);
        float l0 = 0.f, l1 = 0.f;
        auto probs = [&](uint32_t (&r)[32], int ch) {
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float p0 = ex2(fmaf(__uint_as_float(r[2 * j]), c, -mb));
            const float p1 = ex2(fmaf(__uint_as_float(r[2 * j + 1]), c, -mb));
            l0 += p0;
            l1 += p1;
            w[j] = pack2<MBF16>(p0, p1);
          }
          tmem_st16(tS + 16 * ch, w);
        };
#pragma unroll
        for (int ch = 0; ch < 4; ch += 2) {
          tmem_wait_ld(ra);
          tmem_ld32(tS + 32 * (ch + 1), rb);
          if (masked) mask(ra, 32 * ch);
          if (ch == 0) {
            // P of chunk 0 lands on S of chunk 0 only
            probs(ra, 0);
            tmem_wait_ld(rb);
            tmem_ld32(tS + 64, ra);
          } else {
            probs(ra, 2);
            tmem_wait_ld(rb);
          }
          if (masked) mask(rb, 32 * ch + 32);
          probs(rb, ch + 1);
        }
        l += l0 + l1;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&b_p[s]));
      }
      if (!alive) break;
      const long long rec = (static_cast<long long>(sg.seg) * 2 + s);
      if (n > 0) {
        if (!(alive = wait(&b_o[s], oph))) break;
        oph ^= 1u;
        tc_fence_after();
      }
      const bool valid = trow < p.rows;
      if (valid) p.ml[rec * PROWS + row] = make_float2(m == NEG_INF ? NEG_INF : m - BIAS, l);
      if (n > 0) {
        // [D / 4][128 rows][4]: a warp stores 512 contiguous bytes
        float4* dst = reinterpret_cast<float4*>(p.acc + rec * PROWS * D) + row;
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          uint32_t o[32];
          tmem_ld32(tO + d, o);
          tmem_wait_ld(o);
          if (valid) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              dst[(d / 4 + j) * PROWS] = make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]),
                                                     __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3]));
          }
        }
        tc_fence_before();
      }
    }
  } else if (warp < 12) {
    // ============================================================ loaders
    const int lt = tid - 256;
    int stage = 0, pstage = 0, pending = 0;
    uint32_t eph = 1, qph = 1;
    const float sq = p.scale_q != nullptr ? __ldg(p.scale_q) : 1.f;
    const uint32_t flip = sk < 0.f ? 0x80008000u : 0u;  // a negative scale turns Q over: the softmax sees |scale|
    bool alive = true;
    bool withhold = p.inject == 1;
    auto publish = [&]() {  // the oldest unpublished tile is in shared memory
      fence_async_proxy();
      __syncwarp();
      if (lane == 0 && !withhold) mbar_arrive(smem_u32(&b_full[pstage]));
      withhold = false;
      if (++pstage == ST) pstage = 0;
      --pending;
    };
    // page of the tile that this lane looks up
    auto lookup = [&](int tile) -> int {
      const int pg = tile * PPAGES + (lane & 7);
      return pg < p.blocks ? __ldg(p.table + pg) : -1;
    };
    for (long long g = g0; g < g1 && alive;) {
      PrefixSeg sg;
      g += prefix_segment(pl, g, g1, blockIdx.x, &sg);
      bool is_v;
      int tile = sg.t0 + load_item(0, sg.tiles, sg.dual, &is_v);
      int ent = lookup(tile);
      // ---- Q: the unit's row tiles, once the previous segment's products are done
      if (!FP8) {
        cp_async_wait<0>();
        while (pending > 0) publish();
      }
      if (!(alive = wait(&b_qempty, qph))) break;
      qph ^= 1u;
#pragma unroll 1
      for (int s = 0; s < (sg.dual ? 2 : 1); ++s) {
        constexpr int CPR = D / 8;  // 16-byte chunks of a row
#pragma unroll 4
        for (int u = lt; u < PROWS * CPR; u += 128) {
          const int r = u / CPR, ch = u % CPR;
          const int grow = (2 * sg.unit + s) * PROWS + r;
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (grow < p.rows) {
            const int b = grow / p.G, gg = grow - b * p.G;
            x = load_q8<MBF16>(p, b * p.q_b + static_cast<long long>(sg.h * p.G + gg) * p.q_h + ch * 8, sq, flip);
          }
          sts128(sQ + s * C::TILE_BYTES + (ch >> 3) * HALF_BYTES + r * 128 + (((ch & 7) ^ (r & 7)) << 4), x.x, x.y, x.z, x.w);
        }
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&b_qfull));

      // ---- K and V tiles
      if constexpr (!FP8) {
        constexpr int CPR = D / 8, RPS = 128 / CPR;  // chunks of a row, rows per step of the 128 threads
        const int r0 = lt / CPR, ch = lt % CPR;
        for (int idx = 0; idx < 2 * sg.tiles; ++idx) {
          const int t = tile, e = ent;
          const bool v = is_v;
          if (idx + 1 < 2 * sg.tiles) {
            tile = sg.t0 + load_item(idx + 1, sg.tiles, sg.dual, &is_v);
            ent = lookup(tile);
          }
          if (!(alive = wait(&b_empty[stage], eph))) break;
          const char* base = static_cast<const char*>(v ? p.v : p.k);
          const long long sp = (v ? p.vp_p : p.kp_p) * 2, ss = (v ? p.vp_s : p.kp_s) * 2;
          const char* hb = base + (v ? p.vp_h : p.kp_h) * 2 * sg.h + ch * 16;
          const uint32_t dst = sKV + stage * C::TILE_BYTES + (ch >> 3) * HALF_BYTES;
#pragma unroll
          for (int k = 0; k < PTOK / RPS; ++k) {
            const int r = r0 + k * RPS;
            const int ph = __shfl_sync(0xffffffffu, e, (k * RPS) >> 4);
            const bool okp = ph >= 0 && ph < p.num_pages;
            const bool ok = okp && t * PTOK + r < plen;
            if (!okp && t * PTOK + ((k * RPS) & ~15) < plen) s_bad = 1;
            cp_async16_zfill(dst + r * 128 + (((ch & 7) ^ (r & 7)) << 4), ok ? hb + ph * sp + (r & 15) * ss : base, ok);
          }
          cp_async_commit();
          ++pending;
          if (++stage == ST) {
            stage = 0;
            eph ^= 1u;
          }
          if (pending > LOAD_LAG) {
            cp_async_wait<LOAD_LAG>();
            publish();
          }
        }
      } else {
        // e4m3: 16 bytes of a row per load, widened to two 16-byte chunks of f16;
        // the next tile's loads are in flight while this one is widened
        constexpr int NL = 8;  // loads of a thread per tile: 128 rows x 8 chunks / 128
        const int r0 = lt >> 3, ch = lt & 7;
        uint4 buf[NL];
        auto fetch = [&](int t, bool v, int e) {
          const unsigned char* base = static_cast<const unsigned char*>(v ? p.v : p.k);
          const long long sp = v ? p.vp_p : p.kp_p;
          const unsigned char* hb = base + (v ? p.vp_h : p.kp_h) * sg.h + ch * 16 + r0 * (v ? p.vp_s : p.kp_s);
#pragma unroll
          for (int k = 0; k < NL; ++k) {
            const int ph = __shfl_sync(0xffffffffu, e, k);
            const bool okp = ph >= 0 && ph < p.num_pages;
            if (!okp && t * PTOK + k * 16 < plen) s_bad = 1;
            buf[k] = make_uint4(0u, 0u, 0u, 0u);
            if (okp && t * PTOK + k * 16 + r0 < plen) buf[k] = __ldg(reinterpret_cast<const uint4*>(hb + ph * sp));
          }
        };
        fetch(tile, is_v, ent);
        for (int idx = 0; idx < 2 * sg.tiles; ++idx) {
          uint4 cur[NL];
#pragma unroll
          for (int k = 0; k < NL; ++k) cur[k] = buf[k];
          if (idx + 1 < 2 * sg.tiles) {
            tile = sg.t0 + load_item(idx + 1, sg.tiles, sg.dual, &is_v);
            fetch(tile, is_v, lookup(tile));
          }
          if (!(alive = wait(&b_empty[stage], eph))) break;
          const uint32_t dst = sKV + stage * C::TILE_BYTES + (ch >> 2) * HALF_BYTES;
#pragma unroll
          for (int k = 0; k < NL; ++k) {
            const int r = r0 + k * 16;
            uint32_t w[8];
            e4m3x4_to_f16x2x2(cur[k].x, w[0], w[1]);
            e4m3x4_to_f16x2x2(cur[k].y, w[2], w[3]);
            e4m3x4_to_f16x2x2(cur[k].z, w[4], w[5]);
            e4m3x4_to_f16x2x2(cur[k].w, w[6], w[7]);
            const int c0 = (2 * ch) & 7;
            sts128(dst + r * 128 + ((c0 ^ (r & 7)) << 4), w[0], w[1], w[2], w[3]);
            sts128(dst + r * 128 + (((c0 + 1) ^ (r & 7)) << 4), w[4], w[5], w[6], w[7]);
          }
          ++pending;
          publish();
          if (++stage == ST) {
            stage = 0;
            eph ^= 1u;
          }
        }
      }
    }
    cp_async_wait<0>();  // also on the way out after a wait that ran out
    if (alive)
      while (pending > 0) publish();
    if (s_bad && lane == 0 && p.status != nullptr) atomicOr(p.status, FK_STATUS_BAD_PAGE);
  } else if (lane == 0) {
    // ============================================================ MMA issue (one thread)
    constexpr uint32_t idQK = instr_desc(MBF16, PROWS, PTOK, false);
    constexpr uint32_t idPV = instr_desc(MBF16, PROWS, D, true);
    int stage = 0;
    uint32_t fph = 0, qph = 0, pph[2] = {0, 0};
    bool alive = true;
    auto wait1 = [&](uint64_t* bar, uint32_t parity) -> bool {
      if (mbar_wait(smem_u32(bar), parity, p.wait_ns)) return true;
      if (p.status != nullptr) atomicOr(p.status, FK_STATUS_TIMEOUT);
      return false;
    };
    // The tile at the head of the ring: waits for it on its first use, gives it
    // back after its last.
    auto tile_in = [&]() -> bool { return wait1(&b_full[stage], fph); };
    auto tile_out = [&]() {
      mma_commit(smem_u32(&b_empty[stage]));
      if (++stage == ST) {
        stage = 0;
        fph ^= 1u;
      }
    };
    auto qk = [&](int s, int qt, uint32_t k_addr) {
      const uint32_t q_addr = sQ + qt * C::TILE_BYTES;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (k >> 2) * HALF_BYTES + (k & 3) * 32;
        mma_ss(tmem + s * 128, smem_desc(q_addr + off, 16, 1024), smem_desc(k_addr + off, 16, 1024), idQK, k > 0);
      }
      mma_commit(smem_u32(&b_s[s]));
    };
    auto pv = [&](int s, uint32_t v_addr, bool first) {
#pragma unroll
      for (int k = 0; k < PTOK / 16; ++k)
        mma_ts(tmem + 256 + s * D, tmem + s * 128 + 8 * k, smem_desc(v_addr + k * 2048, HALF_BYTES, 1024), idPV,
               !first || k > 0);
    };
    for (long long g = g0; g < g1 && alive;) {
      PrefixSeg sg;
      g += prefix_segment(pl, g, g1, blockIdx.x, &sg);
      const int n = sg.tiles;
      if (!(alive = wait1(&b_qfull, qph))) break;
      qph ^= 1u;
      auto wait_p = [&](int s) -> bool {
        if (!wait1(&b_p[s], pph[s])) return false;
        pph[s] ^= 1u;
        tc_fence_after();
        return true;
      };
      if (sg.dual) {
        // K0: both streams
        if (!(alive = tile_in())) break;
        qk(0, 0, sKV + stage * C::TILE_BYTES);
        qk(1, 1, sKV + stage * C::TILE_BYTES);
        tile_out();
        for (int i = 0; i < n; ++i) {
          // ring: V_i at the head, K_(i+1) behind it
          if (!(alive = tile_in())) break;
          const uint32_t v_addr = sKV + stage * C::TILE_BYTES;
          const int ks = stage + 1 == ST ? 0 : stage + 1;
          const uint32_t kph = stage + 1 == ST ? fph ^ 1u : fph;
          const uint32_t k_addr = sKV + ks * C::TILE_BYTES;
          if (!(alive = wait_p(0))) break;
          pv(0, v_addr, i == 0);
          if (i + 1 < n) {
            if (!(alive = wait1(&b_full[ks], kph))) break;
            qk(0, 0, k_addr);
          } else {
            mma_commit(smem_u32(&b_o[0]));
          }
          if (!(alive = wait_p(1))) break;
          pv(1, v_addr, i == 0);
          tile_out();  // V_i
          if (i + 1 < n) {
            qk(1, 1, k_addr);
            tile_out();  // K_(i+1)
          } else {
            mma_commit(smem_u32(&b_o[1]));
          }
        }
      } else {
        const int pre = min(n, 2);
        for (int s = 0; s < pre && alive; ++s) {
          if (!(alive = tile_in())) break;
          qk(s, 0, sKV + stage * C::TILE_BYTES);
          tile_out();
        }
        for (int i = 0; i < n && alive; ++i) {
          const int s = i & 1;
          if (!(alive = tile_in()) || !(alive = wait_p(s))) break;
          pv(s, sKV + stage * C::TILE_BYTES, i < 2);
          tile_out();
          if (i + 2 < n) {
            if (!(alive = tile_in())) break;
            qk(s, 0, sKV + stage * C::TILE_BYTES);
            tile_out();
          } else {
            mma_commit(smem_u32(&b_o[s]));
          }
        }
      }
      if (!alive) break;
      mma_commit(smem_u32(&b_qempty));
    }
    // nothing of this thread's is in flight when the tensor memory is given back
    mma_commit(smem_u32(&b_drain));
    mbar_wait(smem_u32(&b_drain), 0, p.wait_ns);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------------
// Join: out = (sum_i 2^(m_i - M) acc_i) / (sum_i 2^(m_i - M) l_i [+ 2^(s - M)])
// over the prefix segments of the row and its own part.  Thread = row of a row
// tile, 16 dims; the segments' records are read once, 512 bytes per warp.
// ------------------------------------------------------------------------
struct JoinParams {
  const float2* ml;       // prefix segments
  const float* acc;
  const float2* own_ml;   // [B, QH]
  const float* own_acc;   // [B, QH, D]
  const int* plen_dev;
  int plen, rows, G, kv_heads, q_heads, ctas;
  const float* s_aux;
  const float* scale_v;
  void* out;
  long long o_b, o_h;
  int out_dtype, o_al16;
  const int* own_status;
  int* status;
};

constexpr int JDIMS = 16;

template <int D>
__global__ void __launch_bounds__(PROWS) join_kernel(const __grid_constant__ JoinParams p) {
  grid_dependency_wait();
  grid_dependency_trigger();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && p.status != nullptr && *p.own_status != 0)
    atomicOr(p.status, *p.own_status);
  const int rt = (p.rows + PROWS - 1) / PROWS;
  const int h = blockIdx.x / rt, tile = blockIdx.x % rt;
  const int row = threadIdx.x, grow = tile * PROWS + row;
  if (grow >= p.rows) return;
  const int b = grow / p.G, qh = h * p.G + grow % p.G;
  const int d0 = blockIdx.y * JDIMS;
  const int plen = max(p.plen_dev != nullptr ? __ldg(p.plen_dev) : p.plen, 0);
  const PrefixPlan pl(plen, p.rows, p.kv_heads, p.ctas);
  const int unit = tile >> 1;
  const bool dual = unit < pl.nd;
  int s0 = 0, ns = 0;  // records: stream st of segment s0 + i is record 2 (s0 + i) + st
  if (pl.nt > 0) {
    const long long base = h * pl.gh + pl.unit_base(unit);
    const long long c0 = base / pl.per, c1 = (base + pl.unit_len(unit) - 1) / pl.per;
    s0 = static_cast<int>(c0) + h * pl.upu + unit;
    ns = static_cast<int>(c1 - c0) + 1;
  }
  const int nrec = dual ? ns : 2 * ns;
  auto rec_of = [&](int i) -> long long { return dual ? 2ll * (s0 + i) + (tile & 1) : 2ll * s0 + i; };

  const long long orow = static_cast<long long>(b) * p.q_heads + qh;
  const float2 own = __ldcg(p.own_ml + orow);
  float M = own.x;
  for (int i = 0; i < nrec; ++i) M = fmaxf(M, __ldcg(p.ml + rec_of(i) * PROWS + row).x);
  float L = 0.f;
  if (p.s_aux != nullptr) {
    const float s2 = __ldg(p.s_aux + qh) * LOG2E;
    M = fmaxf(M, s2);
    if (M != NEG_INF) L = exp2f(s2 - M);
  }
  float A[JDIMS];
#pragma unroll
  for (int i = 0; i < JDIMS; ++i) A[i] = 0.f;
  auto add = [&](float e, float4 v, int k) {
    A[4 * k] += e * v.x;
    A[4 * k + 1] += e * v.y;
    A[4 * k + 2] += e * v.z;
    A[4 * k + 3] += e * v.w;
  };
  if (own.x != NEG_INF) {
    const float e = exp2f(own.x - M);
    L += e * own.y;
#pragma unroll
    for (int k = 0; k < JDIMS / 4; ++k) add(e, __ldcg(reinterpret_cast<const float4*>(p.own_acc + orow * D + d0) + k), k);
  }
#pragma unroll 4
  for (int i = 0; i < nrec; ++i) {
    const long long rec = rec_of(i);
    const float2 ml = __ldcg(p.ml + rec * PROWS + row);
    if (ml.x == NEG_INF) continue;  // nothing attended: its accumulators may be unwritten
    const float e = exp2f(ml.x - M);
    L += e * ml.y;
    const float4* src = reinterpret_cast<const float4*>(p.acc + rec * PROWS * D) + (d0 / 4) * PROWS + row;
#pragma unroll
    for (int k = 0; k < JDIMS / 4; ++k) add(e, __ldcg(src + k * PROWS), k);
  }
  const float sv = p.scale_v != nullptr ? __ldg(p.scale_v) : 1.f;
  const long long ob = b * p.o_b + qh * p.o_h + d0;
#pragma unroll
  for (int i = 0; i < JDIMS; ++i) A[i] = norm_out(A[i], 1.f, L, sv);
  const bool bf = p.out_dtype == FK_DTYPE_BF16;
  if (p.o_al16) {
#pragma unroll
    for (int k = 0; k < JDIMS; k += 8) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = bf ? pack2<true>(A[k + 2 * i], A[k + 2 * i + 1]) : pack2<false>(A[k + 2 * i], A[k + 2 * i + 1]);
      *reinterpret_cast<uint4*>(static_cast<unsigned short*>(p.out) + ob + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < JDIMS; ++i) {
      if (bf) static_cast<__nv_bfloat16*>(p.out)[ob + i] = __float2bfloat16_rn(A[i]);
      else static_cast<__half*>(p.out)[ob + i] = __float2half_rn(A[i]);
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

// [own part's decode workspace | own (max, sum) | own acc | prefix (max, sum) | prefix acc]
struct PrefixWs {
  size_t own, own_ml, own_acc, ml, acc, total;
  PrefixWs(int device, int batch, int q_heads, int kv_heads, int head_dim, int kv_dtype) {
    own = fk_decode_workspace_bytes_gqa(device, batch, q_heads, kv_heads, kv_dtype);
    const long long rows = static_cast<long long>(batch) * (q_heads / kv_heads);
    const size_t rt = static_cast<size_t>((rows + PROWS - 1) / PROWS);
    const size_t segs = static_cast<size_t>(prefix_ctas(device)) + static_cast<size_t>(kv_heads) * ((rt + 1) / 2);
    const size_t heads = static_cast<size_t>(batch) * q_heads;
    own_ml = up256(own);
    own_acc = up256(own_ml + heads * sizeof(float2));
    ml = up256(own_acc + heads * head_dim * sizeof(float));
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
      const cudaError_t e = cudaFuncSetAttribute(prefix_kernel<KV, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PCfg<D>::SMEM);
      if (e != cudaSuccess) return fail(FK_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      done[device] = true;
    }
  }
  const cudaError_t e = launch_pdl(prefix_kernel<KV, D>, dim3(ctas), dim3(PTHREADS), PCfg<D>::SMEM, stream, p);
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
  p.zero = reinterpret_cast<int*>(ws);
  p.zero_words = own_part_zero_words(own, w.own);
  p.status = static_cast<int*>(a->status);
  debug_settings(&p.wait_ns, &p.inject);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  DeviceScope scope(device);
  if (kv == FK_DTYPE_F16) rc = D == 64 ? launch_prefix<FK_DTYPE_F16, 64>(p, ctas, device, st) : launch_prefix<FK_DTYPE_F16, 128>(p, ctas, device, st);
  else if (kv == FK_DTYPE_BF16) rc = D == 64 ? launch_prefix<FK_DTYPE_BF16, 64>(p, ctas, device, st) : launch_prefix<FK_DTYPE_BF16, 128>(p, ctas, device, st);
  else rc = launch_prefix<FK_DTYPE_E4M3, 128>(p, ctas, device, st);
  if (rc != FK_OK) return rc;
  rc = own_part_launch(own, reinterpret_cast<float2*>(ws + w.own_ml), reinterpret_cast<float*>(ws + w.own_acc), w.own, st);
  if (rc != FK_OK) return rc;
  JoinParams j = {};
  j.ml = p.ml;
  j.acc = p.acc;
  j.own_ml = reinterpret_cast<const float2*>(ws + w.own_ml);
  j.own_acc = reinterpret_cast<const float*>(ws + w.own_acc);
  j.plen_dev = p.plen_dev;
  j.plen = p.plen;
  j.rows = p.rows;
  j.G = p.G;
  j.kv_heads = KVH;
  j.q_heads = QH;
  j.ctas = ctas;
  j.s_aux = static_cast<const float*>(a->s_aux);
  j.scale_v = kv == FK_DTYPE_E4M3 ? static_cast<const float*>(a->scale_v) : nullptr;
  j.out = a->out;
  j.o_b = a->o_b;
  j.o_h = a->o_h;
  j.out_dtype = static_cast<int>(a->out_dtype);
  j.o_al16 = ((reinterpret_cast<uintptr_t>(a->out) & 15) == 0 && (a->o_b & 7) == 0 && (a->o_h & 7) == 0) ? 1 : 0;
  j.own_status = reinterpret_cast<const int*>(ws);
  j.status = p.status;
  const int rt = (p.rows + PROWS - 1) / PROWS;
  const dim3 grid(static_cast<unsigned>(KVH * rt), static_cast<unsigned>(D / JDIMS));
  const cudaError_t e = D == 128 ? launch_pdl(join_kernel<128>, grid, dim3(PROWS), 0, st, j)
                                 : launch_pdl(join_kernel<64>, grid, dim3(PROWS), 0, st, j);
  return e == cudaSuccess ? FK_OK : fail(FK_ERR_CUDA, "join launch failed: %s", cudaGetErrorString(e));
}
