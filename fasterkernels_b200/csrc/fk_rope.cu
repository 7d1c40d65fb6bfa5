// fk_rope.cu -- per-head RMS norm and position rotation of queries and keys
// in one pass, optionally on the way into a paged KV cache.
//
// For each token t and head row x[D] of q and k, in 32 bits:
//   y = x * rsqrt(mean(x^2) + eps) * w              (with a norm weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)        for the R/2 pairs of the
//   first R dims, pair i being dims (i, i + R/2), or (2i, 2i + 1) interleaved,
//   with cos / sin row position[t] of the tables;
// one rounding, to the output's type: y for q_out / k_out and 16-bit pools,
// y / scale for e4m3 pools.  v rows are copied (or quantised) to their pages.
//
// Every byte is read and written once, so the bound is HBM for many tokens
// and latency for a decode step.  A head row belongs to D / 16 neighbouring
// lanes.  A lane holds two chunks of 8 dims (16 bytes each): 8 dims and their
// 8 partners of the rotation, so that no value changes lanes (dims past R, and
// interleaved pairs, which lie side by side: two adjacent chunks); only the
// mean is reduced across lanes.  The arithmetic runs on packed f32 pairs.
//
// Few tokens: rope_step_kernel, a thread per row part, loads straight to
// registers.  Many: rope_stream_kernel, persistent blocks whose producer warp
// streams whole tokens (rows and table rows) into a shared-memory ring with
// bulk copies, and up to twelve warps that take their rows from there.  A warp
// keeps the same rows of every token, so that kinds and offsets are made once;
// weights and angles are read from shared memory where they are used, since 16
// registers for each spill or cost a block per SM (123 instead of 76 us for the
// append below).
// Measured (device time, inputs past L2): 16384 tokens x 40 heads x 128 bf16
// 58.7 us = 5.9 TB/s (89 % of the copy rate), 116 us with rope_step_kernel; the
// same with v into bf16 pages 72 us = 5.7 TB/s; 6007 x (24 + 4 + 4) heads into
// e4m3 pages 19.3 us = 4.9 TB/s; a step of 32 tokens 2.8 us, 3.9 us with
// rope_stream_kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/fk_decode.h"
#include "fk_f32x2.cuh"
#include "fk_host.h"
#include "fk_prefix.h"
#include "fk_ptx.cuh"

namespace fk {

constexpr int ROPE_THREADS = 128;

// Four 16-bit values <-> two pairs.
template <bool BF>
__device__ __forceinline__ void widen4(uint2 r, f2 (&x)[2]) {
  const uint32_t w[2] = {r.x, r.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (BF) {
      x[i] = mk2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[i] = mk2(f.x, f.y);
    }
  }
}
template <bool BF>
__device__ __forceinline__ uint2 narrow4(const f2 (&x)[2]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float lo, hi;
    split2(x[i], lo, hi);
    w[i] = pack2<BF>(lo, hi);
  }
  return make_uint2(w[0], w[1]);
}

// x / scale saturated to +-448, rounded to nearest e4m3, with the bits that a
// true division gives (as fk_paged_kv_append), nearly always without one: the
// rounded quotient lies between x * lo and x * hi, whose factors are the
// reciprocal made 2^-21 smaller and larger (each of the three roundings on the
// way, and the quotient's own, is off by 2^-24 at most), and rounding to e4m3 is
// monotonic, so where the two ends agree that is the result.  Else (a quotient
// next to the middle of two e4m3 values: 5e-6 of random ones) it divides.  By a
// power of two the product is exact, ties included.  (Dividing always: 23.7
// instead of 19.3 us for 6007 tokens x 32 heads, the k and v warps being late.)
struct Quant {
  float lo, hi;
};
__device__ __forceinline__ float quant_scale(const fk_rope_args& p, int kd) {
  const float* sc = static_cast<const float*>(kd == 1 ? p.scale_k : p.scale_v);
  return sc != nullptr ? __ldg(sc) : 1.f;
}
__device__ __forceinline__ Quant make_quant(const fk_rope_args& p, int kd) {
  const float scale = quant_scale(p, kd);
  const float a = fabsf(scale), r = 1.f / scale;
  const bool pow2 = (__float_as_uint(scale) & 0x7fffffu) == 0;
  Quant q = {pow2 ? r : r * 0.99999952316284f, pow2 ? r : r * 1.00000047683716f};
  if (!(a >= 0x1p-100f && a <= 0x1p100f)) q.lo = -1.f, q.hi = 1.f;  // the reciprocal may leave f32's range: divide
  return q;
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ uint2 quant8(const f2 (&x)[4], const Quant& q, const fk_rope_args& p, int kd) {
  uint32_t a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    split2(mul2(x[i], mk2(q.lo, q.lo)), lo, hi);
    a[i] = e4m3x2(lo, hi);
    split2(mul2(x[i], mk2(q.hi, q.hi)), lo, hi);
    b[i] = e4m3x2(lo, hi);
  }
  uint2 w = make_uint2(a[0] | (a[1] << 16), a[2] | (a[3] << 16));
  if (w.x != (b[0] | (b[1] << 16)) || w.y != (b[2] | (b[3] << 16))) {
    const float scale = quant_scale(p, kd);  // again: registers are short where this is seldom needed
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      split2(i == 0 ? x[0] : i == 1 ? x[1] : i == 2 ? x[2] : x[3], lo, hi);
      const uint32_t d = e4m3x2(lo / scale, hi / scale);
      if (i == 0) w.x = d;
      else if (i == 1) w.x |= d << 16;
      else if (i == 2) w.y = d;
      else w.y |= d << 16;
    }
  }
  return w;
}

// Four consecutive elements of a float / f16 / bf16 array (8-byte aligned).
__device__ __forceinline__ void load4(const void* base, long long i, int dt, f2 (&x)[2]) {
  if (dt == FK_DTYPE_F32) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + i));
    x[0] = mk2(v.x, v.y);
    x[1] = mk2(v.z, v.w);
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(base) + i));
    if (dt == FK_DTYPE_BF16) widen4<true>(v, x);
    else widen4<false>(v, x);
  }
}

template <bool BF>
__device__ __forceinline__ void widen8(uint4 r, f2 (&x)[4]) {
  f2 t[2];
  widen4<BF>(make_uint2(r.x, r.y), t);
  x[0] = t[0];
  x[1] = t[1];
  widen4<BF>(make_uint2(r.z, r.w), t);
  x[2] = t[0];
  x[3] = t[1];
}
template <bool BF>
__device__ __forceinline__ uint4 narrow8(const f2 (&x)[4]) {
  const f2 lo[2] = {x[0], x[1]}, hi[2] = {x[2], x[3]};
  const uint2 a = narrow4<BF>(lo), b = narrow4<BF>(hi);
  return make_uint4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void load8(const void* base, long long i, int dt, f2 (&x)[4]) {
  f2 t[2];
  load4(base, i, dt, t);
  x[0] = t[0];
  x[1] = t[1];
  load4(base, i + 4, dt, t);
  x[2] = t[0];
  x[3] = t[1];
}

// The lane's part of one head row: the norm.  Whole-warp call; `on` says
// whether this row takes part; weight(i) gives the weights of pair i of chunk a
// (i < 4) or b.
template <int D, typename W>
__device__ __forceinline__ void rope_norm(f2 (&xa)[4], f2 (&xb)[4], bool on, float eps, W weight) {
  constexpr int LPH = D / 16;
  f2 ss2 = mul2(xa[0], xa[0]), st2 = mul2(xb[0], xb[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    ss2 = fma2(xa[i], xa[i], ss2);
    st2 = fma2(xb[i], xb[i], st2);
  }
  float s0, s1, s2, s3;
  split2(ss2, s0, s1);
  split2(st2, s2, s3);
  float ss = (s0 + s1) + (s2 + s3);
#pragma unroll
  for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (on) {
    const float inv = rsqrtf(ss * (1.f / D) + eps);
    const f2 inv2 = mk2(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      f2 w0, w1;
      weight(i, w0, w1);
      xa[i] = mul2(mul2(xa[i], inv2), w0);
      xa[i + 1] = mul2(mul2(xa[i + 1], inv2), w1);
      weight(4 + i, w0, w1);
      xb[i] = mul2(mul2(xb[i], inv2), w0);
      xb[i + 1] = mul2(mul2(xb[i + 1], inv2), w1);
    }
  }
}

// The rotation, by cos / sin of the lane's eight pairs.
template <bool IL>
__device__ __forceinline__ void rope_turn(f2 (&xa)[4], f2 (&xb)[4], const f2 (&c)[4], const f2 (&s)[4]) {
  if constexpr (IL) {
    // pairs (2i, 2i + 1): x * (c, c) + swapped x * (-s, s)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f2& x = i < 4 ? xa[i] : xb[i - 4];
      float c0, c1, s0, s1;
      split2(c[i >> 1], c0, c1);
      split2(s[i >> 1], s0, s1);
      const float ci = (i & 1) ? c1 : c0, si = (i & 1) ? s1 : s0;
      x = fma2(swap2(x), mk2(-si, si), mul2(x, mk2(ci, ci)));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f2 a = xa[i], b = xb[i];
      xa[i] = fma2(a, c[i], neg2(mul2(b, s[i])));
      xb[i] = fma2(a, s[i], mul2(b, c[i]));
    }
  }
}

// Store the lane's part: q / k to the dense output, k / v to the page slot.
template <int POOL, bool BF>
__device__ __forceinline__ void rope_store(const fk_rope_args& p, const f2 (&xa)[4], const f2 (&xb)[4], uint4 ra, uint4 rb,
                                           int kd, int head, long long t, int phys, int slot, const Quant& qu, int da, int db) {
  if (kd == 0 || (kd == 1 && p.k_out != nullptr)) {
    unsigned short* dst = kd == 0 ? static_cast<unsigned short*>(p.q_out) + t * p.qo_t + head * p.qo_h
                                  : static_cast<unsigned short*>(p.k_out) + t * p.ko_t + head * p.ko_h;
    *reinterpret_cast<uint4*>(dst + da) = narrow8<BF>(xa);
    *reinterpret_cast<uint4*>(dst + db) = narrow8<BF>(xb);
  }
  if (POOL == 0 || kd == 0 || phys < 0) return;
  const long long o = kd == 1 ? phys * p.kp_p + slot * p.kp_s + head * p.kp_h : phys * p.vp_p + slot * p.vp_s + head * p.vp_h;
  if constexpr (POOL == 2) {
    unsigned char* dst = static_cast<unsigned char*>(kd == 1 ? p.k_pool : p.v_pool) + o;
    *reinterpret_cast<uint2*>(dst + da) = quant8(xa, qu, p, kd);
    *reinterpret_cast<uint2*>(dst + db) = quant8(xb, qu, p, kd);
  } else {
    unsigned short* dst = static_cast<unsigned short*>(kd == 1 ? p.k_pool : p.v_pool) + o;
    *reinterpret_cast<uint4*>(dst + da) = kd == 1 ? narrow8<BF>(xa) : ra;
    *reinterpret_cast<uint4*>(dst + db) = kd == 1 ? narrow8<BF>(xb) : rb;
  }
}

// A token at a position outside the tables: zero rows, nothing appended.
__device__ __forceinline__ void rope_zero(const fk_rope_args& p, int kd, int head, long long t, int da, int db) {
  if (kd > 1 || (kd == 1 && p.k_out == nullptr)) return;
  unsigned short* dst = kd == 0 ? static_cast<unsigned short*>(p.q_out) + t * p.qo_t + head * p.qo_h
                                : static_cast<unsigned short*>(p.k_out) + t * p.ko_t + head * p.ko_h;
  *reinterpret_cast<uint4*>(dst + da) = *reinterpret_cast<uint4*>(dst + db) = make_uint4(0u, 0u, 0u, 0u);
}

// Position of a token, and the page of its slot (-1: none).
template <int POOL>
__device__ __forceinline__ void rope_place(const fk_rope_args& p, long long t, int& pos, int& phys) {
  const int* pos_p = static_cast<const int*>(p.positions);
  const int* seq_p = static_cast<const int*>(p.seq_ids);
  pos = pos_p != nullptr ? __ldg(pos_p + t) : static_cast<int>(t % p.max_pos);
  phys = -1;
  if (POOL) {
    const int seq = seq_p != nullptr ? __ldg(seq_p + t) : static_cast<int>(t);
    const int page = pos >> 4;
    if (pos >= 0 && seq >= 0 && seq < p.table_rows && page < p.max_blocks)
      phys = __ldg(static_cast<const int*>(p.block_table) + seq * p.bt_b + page);
    if (phys >= p.num_pages) phys = -1;
  }
}

template <int POOL>
__device__ __forceinline__ void rope_report(const fk_rope_args& p, bool pos_ok, int phys) {
  if (p.status == nullptr) return;
  if (!pos_ok) atomicOr(static_cast<int*>(p.status), FK_STATUS_BAD_POSITION);
  else if (POOL && phys < 0) atomicOr(static_cast<int*>(p.status), FK_STATUS_BAD_PAGE);
}

// Kind (0 q, 1 k, 2 v, 3 none) and head of row r.
__device__ __forceinline__ void rope_kind(int r, int QH, int KH, int rows, int& kd, int& head) {
  kd = r < QH ? 0 : r < QH + KH ? 1 : r < rows ? 2 : 3;
  head = r - (kd == 0 ? 0 : kd == 1 ? QH : QH + KH);
}

// POOL: 0 none, 1 16-bit, 2 e4m3.  IL: interleaved pairs.  BF: bf16 (else f16).
template <int D, int POOL, bool IL, bool BF>
__global__ void __launch_bounds__(ROPE_THREADS) rope_step_kernel(const __grid_constant__ fk_rope_args p) {
  constexpr int LPH = D / 16;              // lanes per head row
  constexpr int HPP = ROPE_THREADS / LPH;  // head rows of the block
  grid_dependency_wait();
  grid_dependency_trigger();
  const int l = threadIdx.x & (LPH - 1);
  const int QH = static_cast<int>(p.q_heads), KH = static_cast<int>(p.kv_heads);
  const int R = static_cast<int>(p.rotary_dim);
  const bool nq = p.q_weight != nullptr, nk = p.k_weight != nullptr;
  const bool rot = IL ? 16 * l < R : l < R / 16;
  const int da = (!IL && rot) ? 8 * l : 16 * l;  // past R: R + 16 (l - R / 16) = 16 l
  const int db = (!IL && rot) ? R / 2 + 8 * l : da + 8;
  const long long t = blockIdx.x;
  int kd, head;
  rope_kind(blockIdx.y * HPP + threadIdx.x / LPH, QH, KH, QH + (POOL ? 2 : 1) * KH, kd, head);
  uint4 ra = make_uint4(0u, 0u, 0u, 0u), rb = ra;
  if (kd < 3) {
    const unsigned short* src = kd == 0   ? static_cast<const unsigned short*>(p.q) + t * p.q_t + head * p.q_h
                                : kd == 1 ? static_cast<const unsigned short*>(p.k) + t * p.k_t + head * p.k_h
                                          : static_cast<const unsigned short*>(p.v) + t * p.v_t + head * p.v_h;
    ra = *reinterpret_cast<const uint4*>(src + da);
    rb = *reinterpret_cast<const uint4*>(src + db);
  }
  int pos, phys;
  rope_place<POOL>(p, t, pos, phys);
  const bool pos_ok = pos >= 0 && (R == 0 || pos < p.max_pos);
  f2 c[4], s[4];
  if (rot && pos_ok) {
    load8(p.cos, pos * p.cos_row + 8 * l, static_cast<int>(p.table_dtype), c);
    load8(p.sin, pos * p.sin_row + 8 * l, static_cast<int>(p.table_dtype), s);
  }
  f2 wa[4], wb[4];
  const bool norm = kd == 0 ? nq : kd == 1 && nk;
  if (norm) {
    const void* w = kd == 0 ? p.q_weight : p.k_weight;
    const int wt = static_cast<int>(kd == 0 ? p.q_weight_dtype : p.k_weight_dtype);
    load8(w, da, wt, wa);
    load8(w, db, wt, wb);
  }
  if (threadIdx.x == 0 && blockIdx.y == 0) rope_report<POOL>(p, pos_ok, phys);
  Quant qu = {};
  if (POOL == 2) qu = make_quant(p, kd);
  if (!pos_ok) {  // uniform
    rope_zero(p, kd, head, t, da, db);
    return;
  }
  f2 xa[4], xb[4];
  widen8<BF>(ra, xa);
  widen8<BF>(rb, xb);
  if (nq || nk)  // uniform over the grid
    rope_norm<D>(xa, xb, norm, static_cast<float>(p.eps), [&](int i, f2& w0, f2& w1) {
      w0 = i < 4 ? wa[i] : wb[i - 4];
      w1 = i < 4 ? wa[i + 1] : wb[i - 3];
    });
  if (rot && kd < 2) rope_turn<IL>(xa, xb, c, s);
  if (kd < 3) rope_store<POOL, BF>(p, xa, xb, ra, rb, kd, head, t, phys, pos & 15, qu, da, db);
}

// ------------------------------------------------------------------------
// Many tokens.
// ------------------------------------------------------------------------
constexpr int RS_WARPS = 12;                      // most working warps
constexpr int RS_THREADS = (RS_WARPS + 1) * 32;
constexpr int RS_STAGES = 3;
constexpr int RS_TOK = 32;                        // most tokens of a stage

struct RopeStreamParams {
  fk_rope_args a;
  int rows;            // head rows of a token
  int tok;             // tokens of a stage (a power of two)
  int tok_bytes;       // rows * D * 2 + two table rows, rounded to 128
  int table_bytes;     // bytes of a cos (or sin) row
  int contig;          // heads of q, k and v lie one after another
  int wpt, tpw;        // warps that share a token, tokens at work at a time
  unsigned long long wait_ns;
};

// A token's place in the pools (elements; negative: not appended).
struct __align__(16) RopeTok {
  long long k, v;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

template <int D, int POOL, bool IL, bool BF>
__global__ void __launch_bounds__(RS_THREADS, 2) rope_stream_kernel(const __grid_constant__ RopeStreamParams sp) {
  const fk_rope_args& p = sp.a;
  constexpr int LPH = D / 16;
  constexpr int RPW = 32 / LPH;  // head rows of a warp
  constexpr int ROWB = D * 2;
  extern __shared__ __align__(128) unsigned char ring[];
  // Norm weights of q and k, as the lanes of a row read them: their first four
  // dims side by side, their second four, ..  (With dims in order the lanes of a
  // read are 32 bytes apart, two of them on each bank: 61.5 instead of 58.7 us for
  // 16384 tokens x 40 heads.  The same for f32 angles, by reading the halves in
  // turned order, costs selects and registers: 69 us.)
  __shared__ float4 s_w[2][4][LPH];
  __shared__ __align__(8) uint64_t full[RS_STAGES], empty[RS_STAGES];
  __shared__ RopeTok s_tok[RS_STAGES][RS_TOK];
  __shared__ int s_pos[RS_STAGES][RS_TOK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < RS_STAGES; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), sp.wpt * sp.tpw);
    }
    fence_mbar_init();
  }
  __syncthreads();
  grid_dependency_wait();
  grid_dependency_trigger();
  const int QH = static_cast<int>(p.q_heads), KH = static_cast<int>(p.kv_heads);
  const int R = static_cast<int>(p.rotary_dim);
  const int rows = sp.rows, TOK = sp.tok;
  const int stage_bytes = TOK * sp.tok_bytes;
  const bool nq = p.q_weight != nullptr, nk = p.k_weight != nullptr;
  const int workers = sp.wpt * sp.tpw;
  const int nstage = static_cast<int>((p.tokens + TOK - 1) / TOK);  // stages of work (tokens < 2^31 - 2^20)
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    const bool ok = mbar_wait(smem_u32(bar), parity, sp.wait_ns);
    if (__all_sync(0xffffffffu, ok)) return true;
    if (lane == 0 && p.status != nullptr) atomicOr(static_cast<int*>(p.status), FK_STATUS_TIMEOUT);
    return false;
  };

  if (warp == workers) {
    // ---- producer: 32 lanes look up the places of 32 tokens (several stages)
    // at a time, so the chain position -> block table is paid once for them
    const int spb = 32 / TOK;  // stages of a batch
    int stage = 0, n = 0, pos = 0, phys = -1;
    long long koff = -1, voff = -1;
    uint32_t ph = 1, armed = 0, armed_par = 0;
    bool alive = true;
    for (int c = blockIdx.x; c < nstage; c += gridDim.x, ++n) {
      const int sub = n % spb;
      if (sub == 0) {
        const long long t = (static_cast<long long>(c) + lane / TOK * gridDim.x) * TOK + lane % TOK;
        pos = -1;
        koff = voff = -1;
        if (t < p.tokens) {
          rope_place<POOL>(p, t, pos, phys);
          if (pos < 0 || (R > 0 && pos >= p.max_pos)) pos = -1;
          rope_report<POOL>(p, pos >= 0, phys);
          if (POOL && pos >= 0 && phys >= 0) {
            koff = phys * p.kp_p + (pos & 15) * p.kp_s;
            voff = phys * p.vp_p + (pos & 15) * p.vp_s;
          }
        }
      }
      if (!(alive = wait(&empty[stage], ph))) break;
      const int ntok = min(TOK, static_cast<int>(p.tokens) - c * TOK);
      const uint32_t bar = smem_u32(&full[stage]);
      const uint32_t base = smem_u32(ring) + stage * stage_bytes;
      // lane j takes token j of the stage
      const int from = sub * TOK + (lane & (TOK - 1));
      const int tpos = __shfl_sync(0xffffffffu, pos, from);
      const long long tk = __shfl_sync(0xffffffffu, koff, from), tv = __shfl_sync(0xffffffffu, voff, from);
      const bool mine = lane < ntok;
      const unsigned rotated = __ballot_sync(0xffffffffu, mine && R > 0 && tpos >= 0);
      if (mine) {
        s_pos[stage][lane] = tpos;
        s_tok[stage][lane] = RopeTok{tk, tv};
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(bar, ntok * rows * ROWB + __popc(rotated) * 2 * sp.table_bytes);
      armed |= 1u << stage;
      armed_par = (armed_par & ~(1u << stage)) | ((ph ^ 1u) << stage);
      __syncwarp();
      if (mine) {
        const long long t = c * TOK + lane;
        const uint32_t dst = base + lane * sp.tok_bytes;
        if ((rotated >> lane) & 1u) {
          const int es = p.table_dtype == FK_DTYPE_F32 ? 4 : 2;
          bulk_load(dst + rows * ROWB, static_cast<const char*>(p.cos) + tpos * p.cos_row * es, sp.table_bytes, bar);
          bulk_load(dst + rows * ROWB + sp.table_bytes, static_cast<const char*>(p.sin) + tpos * p.sin_row * es,
                    sp.table_bytes, bar);
        }
        if (sp.contig) {
          bulk_load(dst, static_cast<const unsigned short*>(p.q) + t * p.q_t, QH * ROWB, bar);
          bulk_load(dst + QH * ROWB, static_cast<const unsigned short*>(p.k) + t * p.k_t, KH * ROWB, bar);
          if (POOL) bulk_load(dst + (QH + KH) * ROWB, static_cast<const unsigned short*>(p.v) + t * p.v_t, KH * ROWB, bar);
        }
      }
      if (!sp.contig) {
        for (int i = lane; i < ntok * rows; i += 32) {
          const int j = i / rows, r = i - j * rows;
          const long long t = c * TOK + j;
          int kd, head;
          rope_kind(r, QH, KH, rows, kd, head);
          const unsigned short* src = kd == 0   ? static_cast<const unsigned short*>(p.q) + t * p.q_t + head * p.q_h
                                      : kd == 1 ? static_cast<const unsigned short*>(p.k) + t * p.k_t + head * p.k_h
                                                : static_cast<const unsigned short*>(p.v) + t * p.v_t + head * p.v_h;
          bulk_load(base + j * sp.tok_bytes + r * ROWB, src, ROWB, bar);
        }
      }
      if (++stage == RS_STAGES) {
        stage = 0;
        ph ^= 1u;
      }
    }
    // a wait ran out: let the copies in flight land before the block exits
    if (!alive && lane == 0)
      for (int i = 0; i < RS_STAGES; ++i)
        if ((armed >> i) & 1u) mbar_wait(smem_u32(&full[i]), (armed_par >> i) & 1u, sp.wait_ns);
    return;
  }

  // ---- workers: warp w takes the groups of RPW rows w % wpt, + wpt, .. of the
  // tokens w / wpt, + tpw, .. of a stage
  for (int i = threadIdx.x; i < 2 * (D / 4); i += workers * 32) {
    const int kind = i / (D / 4), piece = i % (D / 4) / LPH, wl = i % LPH;
    const void* w = kind == 0 ? p.q_weight : p.k_weight;
    if (w == nullptr) continue;
    const bool turned = !IL && wl < R / 16;  // the dims of a lane: see da, db
    const int at = (piece < 2 ? (turned ? 8 * wl : 16 * wl) : (turned ? R / 2 + 8 * wl : 16 * wl + 8)) + 4 * (piece & 1);
    f2 x[2];
    load4(w, at, static_cast<int>(kind == 0 ? p.q_weight_dtype : p.k_weight_dtype), x);
    float4 f;
    split2(x[0], f.x, f.y);
    split2(x[1], f.z, f.w);
    s_w[kind][piece][wl] = f;
  }
  named_bar_sync(1, workers * 32);
  const int l = lane & (LPH - 1);
  const bool rot = IL ? 16 * l < R : l < R / 16;
  const int da = (!IL && rot) ? 8 * l : 16 * l;
  const int db = (!IL && rot) ? R / 2 + 8 * l : da + 8;
  const float eps = static_cast<float>(p.eps);
  const int tdt = static_cast<int>(p.table_dtype);
  const int tw = warp / sp.wpt, gw = warp - tw * sp.wpt;
  const int gpt = (rows + RPW - 1) / RPW;
  const uint32_t ring0 = smem_u32(ring);

  // of the lane's current row
  int kd = 3;
  uint32_t off = 0;                 // in a token's shared memory
  unsigned short* dense = nullptr;  // row of token 0 in its 16-bit output, or null
  long long dense_t = 0;
  char* page = nullptr;             // row of slot 0 of page 0 in its pool, or null
  bool norm = false;
  uint32_t wts = 0;                 // its weights
  Quant qu = {};
  auto row = [&](int g) {
    const int r = g * RPW + lane / LPH;
    int head;
    rope_kind(r, QH, KH, rows, kd, head);
    off = (r < rows ? r : 0) * ROWB;
    dense = nullptr;
    if (kd == 0) {
      dense = static_cast<unsigned short*>(p.q_out) + head * p.qo_h;
      dense_t = p.qo_t;
    } else if (kd == 1 && p.k_out != nullptr) {
      dense = static_cast<unsigned short*>(p.k_out) + head * p.ko_h;
      dense_t = p.ko_t;
    }
    page = nullptr;
    if (POOL && kd == 1) page = static_cast<char*>(p.k_pool) + head * p.kp_h * (POOL == 2 ? 1 : 2);
    if (POOL && kd == 2) page = static_cast<char*>(p.v_pool) + head * p.vp_h * (POOL == 2 ? 1 : 2);
    norm = kd == 0 ? nq : kd == 1 && nk;
    wts = smem_u32(&s_w[kd == 0 ? 0 : 1][0][l]);
    if (POOL == 2) qu = make_quant(p, kd);
  };
  row(gw);
  int stage = 0;
  uint32_t ph = 0;
  for (int c = blockIdx.x; c < nstage; c += gridDim.x) {
    if (!wait(&full[stage], ph)) break;
    const int t0 = c * TOK;
    const int ntok = min(TOK, static_cast<int>(p.tokens) - t0);
    for (int j = tw; j < ntok; j += sp.tpw) {
      const uint32_t base = ring0 + stage * stage_bytes + j * sp.tok_bytes;
      const int pos = s_pos[stage][j];
      for (int g = gw; g < gpt; g += sp.wpt) {
        if (gpt > sp.wpt) row(g);
        unsigned short* dst = dense + (t0 + j) * dense_t;
        if (pos < 0) {  // outside the tables: zero rows, nothing appended
          if (dense != nullptr)
            *reinterpret_cast<uint4*>(dst + da) = *reinterpret_cast<uint4*>(dst + db) = make_uint4(0u, 0u, 0u, 0u);
          continue;
        }
        f2 xa[4], xb[4];
        widen8<BF>(lds128(base + off + da * 2), xa);
        widen8<BF>(lds128(base + off + db * 2), xb);
        if (nq || nk)  // uniform over the grid
          rope_norm<D>(xa, xb, norm, eps, [&](int i, f2& w0, f2& w1) {
            const uint4 w = lds128(wts + (i / 2) * (LPH * 16));
            w0 = mk2(__uint_as_float(w.x), __uint_as_float(w.y));
            w1 = mk2(__uint_as_float(w.z), __uint_as_float(w.w));
          });
        if (rot && kd < 2) {
          f2 cs[4], sn[4];
          const uint32_t tc = base + rows * ROWB;
          if (tdt == FK_DTYPE_F32) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint4 x = lds128(tc + 32 * l + 16 * i), y = lds128(tc + sp.table_bytes + 32 * l + 16 * i);
              cs[2 * i] = mk2(__uint_as_float(x.x), __uint_as_float(x.y));
              cs[2 * i + 1] = mk2(__uint_as_float(x.z), __uint_as_float(x.w));
              sn[2 * i] = mk2(__uint_as_float(y.x), __uint_as_float(y.y));
              sn[2 * i + 1] = mk2(__uint_as_float(y.z), __uint_as_float(y.w));
            }
          } else {
            const uint4 x = lds128(tc + 16 * l), y = lds128(tc + sp.table_bytes + 16 * l);
            if (tdt == FK_DTYPE_BF16) {
              widen8<true>(x, cs);
              widen8<true>(y, sn);
            } else {
              widen8<false>(x, cs);
              widen8<false>(y, sn);
            }
          }
          rope_turn<IL>(xa, xb, cs, sn);
        }
        if (dense != nullptr) {
          *reinterpret_cast<uint4*>(dst + da) = narrow8<BF>(xa);
          *reinterpret_cast<uint4*>(dst + db) = narrow8<BF>(xb);
        }
        if (POOL && page != nullptr) {
          const long long at = kd == 1 ? s_tok[stage][j].k : s_tok[stage][j].v;
          if (at >= 0) {
            if constexpr (POOL == 2) {
              *reinterpret_cast<uint2*>(page + at + da) = quant8(xa, qu, p, kd);
              *reinterpret_cast<uint2*>(page + at + db) = quant8(xb, qu, p, kd);
            } else if (kd == 1) {
              *reinterpret_cast<uint4*>(page + 2 * (at + da)) = narrow8<BF>(xa);
              *reinterpret_cast<uint4*>(page + 2 * (at + db)) = narrow8<BF>(xb);
            } else {  // v as it is
              *reinterpret_cast<uint4*>(page + 2 * (at + da)) = lds128(base + off + da * 2);
              *reinterpret_cast<uint4*>(page + 2 * (at + db)) = lds128(base + off + db * 2);
            }
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&empty[stage]));
    if (++stage == RS_STAGES) {
      stage = 0;
      ph ^= 1u;
    }
  }
}

constexpr int RS_MAX_SMEM = 200 * 1024;
constexpr int RS_STAGE_BYTES = 26 * 1024;  // tokens are gathered up to this
constexpr int RS_MIN_STAGES = 3;           // of a block (fewer: rope_step_kernel)

template <int D, int POOL, bool IL, bool BF>
cudaError_t launch_rope(const fk_rope_args& a, int device, cudaStream_t stream) {
  const long long rows = a.q_heads + (POOL ? 2 : 1) * a.kv_heads;
  const int table_bytes = static_cast<int>(a.rotary_dim / 2 * (a.table_dtype == FK_DTYPE_F32 ? 4 : 2));
  const long long tok_bytes = (rows * D * 2 + 2 * table_bytes + 127) / 128 * 128;
  constexpr int HPP = ROPE_THREADS / (D / 16);
  // Warps of a token: its groups of rows in as few rounds as RS_WARPS allow.
  const int gpt = static_cast<int>((rows + HPP / 4 - 1) / (HPP / 4));
  const int rounds = (gpt + RS_WARPS - 1) / RS_WARPS;
  const int wpt = (gpt + rounds - 1) / rounds;
  if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
  static int sms[64] = {};
  if (sms[device] == 0) {
    cudaError_t e = cudaFuncSetAttribute(rope_stream_kernel<D, POOL, IL, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, RS_MAX_SMEM);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms[device], cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return e;
  }
  // A block wants some stages to stream: stages of as many tokens as fit, of
  // fewer where that leaves blocks with less than RS_MIN_STAGES.  (4099 tokens x
  // 15 heads x 64: 6.2 us so, 8.2 with rope_step_kernel, which 26 KB stages and
  // two of them a block would choose; 1200 x 40 x 128: 7.2 us, 7.8 with two.  With
  // one, 300 x 48 x 128 takes 4.9 us, 3.8 with rope_step_kernel.)
  int tok = 1, tpw = 1, threads = 0;
  while (tok < RS_TOK && 2 * tok * tok_bytes <= RS_STAGE_BYTES) tok *= 2;
  long long smem = 0, grid = 0, work = 0;
  bool stream_ok = false;
  for (; tok >= 1 && !stream_ok && a.tokens <= 0x7fe00000; tok /= 2) {
    smem = RS_STAGES * tok * tok_bytes;
    work = (a.tokens + tok - 1) / tok;
    if (smem > RS_MAX_SMEM || work < 2 * sms[device]) continue;
    tpw = RS_WARPS / wpt < tok ? RS_WARPS / wpt : tok;
    threads = (wpt * tpw + 1) * 32;
    int fit = 0;  // blocks that share an SM
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, rope_stream_kernel<D, POOL, IL, BF>, threads, static_cast<size_t>(smem));
    grid = static_cast<long long>(sms[device]) * fit;
    stream_ok = fit > 0 && work >= RS_MIN_STAGES * grid;
    if (stream_ok) break;
  }
  if (!stream_ok)
    return launch_pdl(rope_step_kernel<D, POOL, IL, BF>,
                      dim3(static_cast<unsigned>(a.tokens), static_cast<unsigned>((rows + HPP - 1) / HPP)),
                      dim3(ROPE_THREADS), 0, stream, a);
  RopeStreamParams sp;
  sp.a = a;
  sp.rows = static_cast<int>(rows);
  sp.tok = tok;
  sp.tok_bytes = static_cast<int>(tok_bytes);
  sp.table_bytes = table_bytes;
  sp.contig = (a.q_h == D || a.q_heads == 1) && (a.k_h == D || a.kv_heads == 1) && (!POOL || a.v_h == D || a.kv_heads == 1);
  sp.wpt = wpt;
  sp.tpw = tpw;
  int inject;
  debug_settings(&sp.wait_ns, &inject);
  return launch_pdl(rope_stream_kernel<D, POOL, IL, BF>, dim3(static_cast<unsigned>(work < grid ? work : grid)),
                    dim3(threads), static_cast<size_t>(smem), stream, sp);
}

template <int D>
cudaError_t launch_rope_d(const fk_rope_args& a, int device, cudaStream_t stream) {
  const int pool = a.k_pool == nullptr ? 0 : a.pool_dtype == FK_DTYPE_E4M3 ? 2 : 1;
  const bool il = a.interleaved != 0, bf = a.dtype == FK_DTYPE_BF16;
#define FK_ROPE(P) \
  (il ? (bf ? launch_rope<D, P, true, true>(a, device, stream) : launch_rope<D, P, true, false>(a, device, stream)) \
      : (bf ? launch_rope<D, P, false, true>(a, device, stream) : launch_rope<D, P, false, false>(a, device, stream)))
  return pool == 0 ? FK_ROPE(0) : pool == 1 ? FK_ROPE(1) : FK_ROPE(2);
#undef FK_ROPE
}

namespace {

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int rope_checks(const fk_rope_args& a) {
  if (a.q == nullptr || a.k == nullptr || a.q_out == nullptr)
    return fail(FK_ERR_INVALID_ARG, "q, k and q_out must be non-null");
  if (a.tokens < 0 || a.q_heads <= 0 || a.kv_heads <= 0)
    return fail(FK_ERR_INVALID_ARG, "bad sizes");
  if (a.tokens > 0x7fffffffLL || a.q_heads > 65535 || a.kv_heads > 65535) return fail(FK_ERR_INVALID_ARG, "sizes too large");
  if (a.head_dim != 128 && a.head_dim != 64)
    return fail(FK_ERR_UNSUPPORTED, "head_dim must be 128 or 64 (got %lld)", static_cast<long long>(a.head_dim));
  if (a.dtype != FK_DTYPE_F16 && a.dtype != FK_DTYPE_BF16) return fail(FK_ERR_UNSUPPORTED, "q, k and v must be f16 or bf16");
  if (a.rotary_dim < 0 || a.rotary_dim > a.head_dim || a.rotary_dim % 16 != 0)
    return fail(FK_ERR_UNSUPPORTED, "rotary_dim must be a multiple of 16 up to head_dim (got %lld)",
                static_cast<long long>(a.rotary_dim));
  if (a.rotary_dim > 0) {
    if (a.cos == nullptr || a.sin == nullptr) return fail(FK_ERR_INVALID_ARG, "cos and sin must be non-null");
    if (a.max_pos <= 0) return fail(FK_ERR_INVALID_ARG, "the cos / sin tables must have rows");
    if (a.table_dtype != FK_DTYPE_F32 && a.table_dtype != FK_DTYPE_F16 && a.table_dtype != FK_DTYPE_BF16)
      return fail(FK_ERR_UNSUPPORTED, "cos / sin must be f32, f16 or bf16");
    const int es = a.table_dtype == FK_DTYPE_F32 ? 4 : 2;
    if (!al16(a.cos) || !al16(a.sin) || ((a.cos_row | a.sin_row) * es) % 16 != 0)
      return fail(FK_ERR_INVALID_ARG, "cos / sin rows must be 16-byte aligned");
  }
  if (a.positions == nullptr && (a.rotary_dim == 0 || a.k_pool != nullptr))
    return fail(FK_ERR_INVALID_ARG, "positions must be non-null");
  for (int i = 0; i < 2; ++i) {
    const void* w = i == 0 ? a.q_weight : a.k_weight;
    const int64_t wd = i == 0 ? a.q_weight_dtype : a.k_weight_dtype;
    if (w == nullptr) continue;
    if (wd != FK_DTYPE_F32 && wd != FK_DTYPE_F16 && wd != FK_DTYPE_BF16)
      return fail(FK_ERR_UNSUPPORTED, "norm weights must be f32, f16 or bf16");
    if (!al16(w)) return fail(FK_ERR_INVALID_ARG, "norm weights must be 16-byte aligned");
  }
  if (((a.q_t | a.q_h | a.k_t | a.k_h | a.qo_t | a.qo_h | a.ko_t | a.ko_h) * 2) % 16 != 0)
    return fail(FK_ERR_INVALID_ARG, "strides must be multiples of 16 bytes");
  if (!al16(a.q) || !al16(a.k) || !al16(a.q_out) || !al16(a.k_out))
    return fail(FK_ERR_INVALID_ARG, "tensors must be 16-byte aligned");
  if (a.k_pool == nullptr) {
    if (a.k_out == nullptr) return fail(FK_ERR_INVALID_ARG, "k_out must be non-null without a pool");
    return FK_OK;
  }
  if (a.v == nullptr || a.v_pool == nullptr || a.block_table == nullptr)
    return fail(FK_ERR_INVALID_ARG, "v, v_pool and block_table must be non-null with a pool");
  if (a.num_pages <= 0 || a.num_pages > 0x7fffffffLL || a.max_blocks < 0 || a.table_rows < 0)
    return fail(FK_ERR_INVALID_ARG, "bad pool sizes");
  if (a.pool_dtype != FK_DTYPE_E4M3 && a.pool_dtype != a.dtype)
    return fail(FK_ERR_INVALID_ARG, "a 16-bit pool must have the dtype of the new K/V");
  const int es = a.pool_dtype == FK_DTYPE_E4M3 ? 1 : 2;
  if (((a.kp_p | a.kp_h | a.kp_s | a.vp_p | a.vp_h | a.vp_s) * es) % 16 != 0 || ((a.v_t | a.v_h) * 2) % 16 != 0)
    return fail(FK_ERR_INVALID_ARG, "strides must be multiples of 16 bytes");
  if (!al16(a.v) || !al16(a.k_pool) || !al16(a.v_pool))
    return fail(FK_ERR_INVALID_ARG, "tensors must be 16-byte aligned");
  return FK_OK;
}

}  // namespace
}  // namespace fk

using namespace fk;

extern "C" int fk_qk_norm_rope(const fk_rope_args* args, void* stream) {
  if (args == nullptr) return fail(FK_ERR_INVALID_ARG, "args must be non-null");
  if (args->tokens == 0) return FK_OK;
  int rc = rope_checks(*args);
  if (rc != FK_OK) return rc;
  int device = 0;
  if ((rc = pointer_device(args->q, "q", &device)) != FK_OK) return rc;
  DeviceScope scope(device);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = args->head_dim == 128 ? launch_rope_d<128>(*args, device, st) : launch_rope_d<64>(*args, device, st);
  if (e != cudaSuccess) return fail(FK_ERR_CUDA, "rope launch failed: %s", cudaGetErrorString(e));
  return FK_OK;
}
