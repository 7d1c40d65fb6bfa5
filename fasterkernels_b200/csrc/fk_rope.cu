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
// and latency for a decode step.  A head row is held by D / 8 neighbouring
// lanes, 8 dims (16 bytes) each; the mean is a shuffle reduction over them and
// the half-split partner comes from another lane of the row, so nothing goes
// through shared memory.  All heads of a token run in one block (a thread
// keeps its 8 dims, hence its cos / sin, for every head it visits) unless the
// tokens alone do not fill the GPU.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/fk_decode.h"
#include "fk_host.h"
#include "fk_ptx.cuh"

namespace fk {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_UNROLL = 4;  // head rows a thread loads before it works on the first

__device__ __forceinline__ void widen8(uint4 r, int dt, float (&x)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dt == FK_DTYPE_BF16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

__device__ __forceinline__ uint4 narrow8(const float (&x)[8], int dt) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = dt == FK_DTYPE_BF16 ? pack2<true>(x[2 * i], x[2 * i + 1]) : pack2<false>(x[2 * i], x[2 * i + 1]);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// x / scale saturated to +-448, rounded to nearest e4m3 (a true division, as
// fk_paged_kv_append)
__device__ __forceinline__ uint2 quant8(const float (&x)[8], float scale) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    w[i >> 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x[i] / scale, x[i + 1] / scale),
                                                                 __NV_SATFINITE, __NV_E4M3))
                 << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}

// N consecutive elements of a float / f16 / bf16 array as floats (16-byte
// aligned for N = 8, 8-byte for N = 4 of the 16-bit types).
template <int N>
__device__ __forceinline__ void load_as_float(const void* base, long long i, int dt, float* x) {
  if (dt == FK_DTYPE_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      const float4 v = __ldg(p + k);
      x[4 * k] = v.x;
      x[4 * k + 1] = v.y;
      x[4 * k + 2] = v.z;
      x[4 * k + 3] = v.w;
    }
  } else {
    const uint2* p = reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(base) + i);
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      const uint2 v = __ldg(p + k);
      const uint32_t w[2] = {v.x, v.y};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (dt == FK_DTYPE_BF16) {
          x[4 * k + 2 * j] = __uint_as_float(w[j] << 16);
          x[4 * k + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          x[4 * k + 2 * j] = f.x;
          x[4 * k + 2 * j + 1] = f.y;
        }
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const __grid_constant__ fk_rope_args p) {
  constexpr int LPH = D / 8;                 // lanes per head row
  constexpr int HPP = ROPE_THREADS / LPH;    // head rows per pass of the block
  grid_dependency_wait();
  grid_dependency_trigger();
  const long long t = blockIdx.x;
  const int l = threadIdx.x & (LPH - 1);
  const int d0 = l * 8;
  const int dt = static_cast<int>(p.dtype);
  const int QH = static_cast<int>(p.q_heads), KH = static_cast<int>(p.kv_heads);
  const bool paged = p.k_pool != nullptr;
  const int rows = QH + (paged ? 2 : 1) * KH;

  // position, and the page slot of the token
  const int* pos_p = static_cast<const int*>(p.positions);
  const long long pos = pos_p != nullptr ? static_cast<long long>(pos_p[t]) : t % p.max_pos;
  const int R = static_cast<int>(p.rotary_dim);
  const bool pos_ok = pos >= 0 && (R == 0 || pos < p.max_pos);
  int phys = -1;
  if (paged && pos_ok) {
    const int* sp = static_cast<const int*>(p.seq_ids);
    const long long seq = sp != nullptr ? static_cast<long long>(sp[t]) : t;
    const long long page = pos >> 4;
    if (seq >= 0 && seq < p.table_rows && page < p.max_blocks)
      phys = static_cast<const int*>(p.block_table)[seq * p.bt_b + page];
    if (phys >= p.num_pages) phys = -1;
  }
  if (threadIdx.x == 0 && blockIdx.y == 0 && p.status != nullptr) {
    if (!pos_ok) atomicOr(static_cast<int*>(p.status), FK_STATUS_BAD_POSITION);
    else if (paged && phys < 0) atomicOr(static_cast<int*>(p.status), FK_STATUS_BAD_PAGE);
  }
  const int slot = static_cast<int>(pos & 15);

  // this thread's cos / sin: of dims d0 .. d0 + 7 (half-split) or of the four
  // pairs in them (interleaved)
  float cs[8], sn[8];
  const int half = R / 2;
  const int hl = half / 8;  // lanes of a half
  const bool rot = pos_ok && d0 < R;
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = 1.f, sn[i] = 0.f;
  if (rot) {
    const int tdt = static_cast<int>(p.table_dtype);
    if (p.interleaved) {
      load_as_float<4>(p.cos, pos * p.cos_row + 4 * l, tdt, cs);
      load_as_float<4>(p.sin, pos * p.sin_row + 4 * l, tdt, sn);
    } else {
      const int j = l < hl ? d0 : d0 - half;
      load_as_float<8>(p.cos, pos * p.cos_row + j, tdt, cs);
      load_as_float<8>(p.sin, pos * p.sin_row + j, tdt, sn);
    }
  }
  // lane of the row that holds the partner dims (half-split)
  const int lane = threadIdx.x & 31;
  const int partner = (lane - l) + (l < hl ? l + hl : (l < 2 * hl ? l - hl : l));

  const float eps = static_cast<float>(p.eps);
  const float sk = p.scale_k != nullptr ? __ldg(static_cast<const float*>(p.scale_k)) : 1.f;
  const float sv = p.scale_v != nullptr ? __ldg(static_cast<const float*>(p.scale_v)) : 1.f;
  const int pdt = static_cast<int>(p.pool_dtype);

  // blockIdx.y takes every gridDim.y-th pass
  const int step = HPP * gridDim.y * ROPE_UNROLL;
  const int r00 = blockIdx.y * HPP + threadIdx.x / LPH;
  // every lane runs every round: the shuffles are warp-wide
  for (int base = 0; base < rows; base += step) {
    uint4 raw[ROPE_UNROLL];
#pragma unroll
    for (int u = 0; u < ROPE_UNROLL; ++u) {
      const int r = base + r00 + u * HPP * static_cast<int>(gridDim.y);
      raw[u] = make_uint4(0u, 0u, 0u, 0u);
      if (r < QH)
        raw[u] = *reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p.q) + t * p.q_t + r * p.q_h + d0);
      else if (r < QH + KH)
        raw[u] = *reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p.k) + t * p.k_t + (r - QH) * p.k_h + d0);
      else if (r < rows)
        raw[u] = *reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p.v) + t * p.v_t +
                                                 (r - QH - KH) * p.v_h + d0);
    }
#pragma unroll
    for (int u = 0; u < ROPE_UNROLL; ++u) {
      if (base + u * HPP * static_cast<int>(gridDim.y) >= rows) break;  // uniform over the block
      const int r = base + r00 + u * HPP * static_cast<int>(gridDim.y);
      float x[8];
      widen8(raw[u], dt, x);
      const bool is_q = r < QH, is_k = !is_q && r < QH + KH;
      const void* w = is_q ? p.q_weight : is_k ? p.k_weight : nullptr;
      if (p.q_weight != nullptr || p.k_weight != nullptr) {  // uniform
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w != nullptr) {
          const float inv = rsqrtf(ss * (1.f / D) + eps);
          float wt[8];
          load_as_float<8>(w, d0, static_cast<int>(is_q ? p.q_weight_dtype : p.k_weight_dtype), wt);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * wt[i];
        }
      }
      if (R > 0) {  // uniform
        if (p.interleaved) {
          if (rot && (is_q || is_k)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float a = x[2 * i], b = x[2 * i + 1];
              x[2 * i] = a * cs[i] - b * sn[i];
              x[2 * i + 1] = b * cs[i] + a * sn[i];
            }
          }
        } else {
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], partner);
          if (rot && (is_q || is_k)) {
            const float sg = l < hl ? -1.f : 1.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * cs[i] + sg * (y[i] * sn[i]);
          }
        }
      }
      if (r >= rows) continue;
      if (is_q) {
        *reinterpret_cast<uint4*>(static_cast<unsigned short*>(p.q_out) + t * p.qo_t + r * p.qo_h + d0) =
            pos_ok ? narrow8(x, dt) : make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      const int h = is_k ? r - QH : r - QH - KH;
      if (is_k && p.k_out != nullptr)
        *reinterpret_cast<uint4*>(static_cast<unsigned short*>(p.k_out) + t * p.ko_t + h * p.ko_h + d0) =
            pos_ok ? narrow8(x, dt) : make_uint4(0u, 0u, 0u, 0u);
      if (phys < 0) continue;
      const long long o = is_k ? phys * p.kp_p + h * p.kp_h + slot * p.kp_s + d0
                               : phys * p.vp_p + h * p.vp_h + slot * p.vp_s + d0;
      void* pool = is_k ? p.k_pool : p.v_pool;
      if (pdt == FK_DTYPE_E4M3)
        *reinterpret_cast<uint2*>(static_cast<unsigned char*>(pool) + o) = quant8(x, is_k ? sk : sv);
      else
        *reinterpret_cast<uint4*>(static_cast<unsigned short*>(pool) + o) = is_k ? narrow8(x, dt) : raw[u];
    }
  }
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
  const int rows = static_cast<int>(args->q_heads + (args->k_pool != nullptr ? 2 : 1) * args->kv_heads);
  const int hpp = ROPE_THREADS / static_cast<int>(args->head_dim / 8);
  const int passes = (rows + hpp - 1) / hpp;
  // Few tokens: one block per pass of a token (shorter chains per thread).
  const int ny = args->tokens < 512 ? (passes < 65535 ? passes : 65535) : 1;
  const dim3 grid(static_cast<unsigned>(args->tokens), static_cast<unsigned>(ny));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = args->head_dim == 128 ? launch_pdl(rope_kernel<128>, grid, dim3(ROPE_THREADS), 0, st, *args)
                                              : launch_pdl(rope_kernel<64>, grid, dim3(ROPE_THREADS), 0, st, *args);
  if (e != cudaSuccess) return fail(FK_ERR_CUDA, "rope launch failed: %s", cudaGetErrorString(e));
  return FK_OK;
}
