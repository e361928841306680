// Norms of queries and keys for each head, rotary positions, and the paged K/V append, in one pass over the QKV
// projection's rows. For a head vector x of d values at position p:
//   y = x * rsqrt(mean(x^2) + eps) * w          (q and k heads, where a weight is given)
//   z_j = y_j cos_j - y_{j+d/2} sin_j,  z_{j+d/2} = y_{j+d/2} cos_j + y_j sin_j   (q and k heads, where a table is)
// q goes out in bf16 or fp32, K and V into their slot of the pools in bf16, or as int8 codes with one scale per
// vector: s = max(max|z| / 127, 1e-8), code = clamp(round_half_even(z / s), -128, 127). An infinity or NaN in z makes s one:
// the whole vector then reads back as NaN.
//
// Bound by memory: every value is read once and written once. d / 8 lanes hold a head, each with four adjacent
// values of the first half and their four rotation partners of the second, so that loads are 16 bytes, the
// rotation needs no exchange, and a norm or an absolute maximum is a few shuffles. All sums are fp32; the one
// rounding is the store (q and K/V feed bf16 tensor-core products).
// Two heads per group of lanes keep enough loads in flight: 8192 rows of 24/8 heads of 128 take 48 us on a B200, 5.3 TB/s
// of the 6.55 that a copy reaches (56 us with one head and the loads behind the slot's); 160 rows 5 us, the launch.
#include "common.cuh"

namespace {

constexpr int kAppThreads = 256;
constexpr int kUnits = 2;  // heads per group of lanes

struct AppendArgs {
  const void* qkv;
  int64_t ld, rows;
  const int32_t *positions, *slots;
  const float *cos_sin, *qw, *kw;
  float eps;
  int max_pos, hq, hkv;
  void* q_out;
  void *k_pool, *v_pool;
  float *k_scales, *v_scales;
  int64_t num_blocks;
};

template <bool B16>
__device__ __forceinline__ float4 load4(const void* base, int64_t i) {
  if constexpr (B16) {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + i);
    return make_float4(bf16lo(v.x), bf16hi(v.x), bf16lo(v.y), bf16hi(v.y));
  } else {
    return *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
  }
}

__device__ __forceinline__ void store4_bf16(__nv_bfloat16* p, const float4& a) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
}

// The larger of two, or NaN where either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Codes of four values. A quotient that is NaN has code 0: beside the scale that it has then (NaN, or infinite), any value of
// the vector reads back as NaN.
__device__ __forceinline__ uint32_t code4(const float4& a, float s) {
  const float v[4] = {a.x, a.y, a.z, a.w};
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = min(max(__float2int_rn(__fdiv_rn(v[i], s)), -128), 127);
    w |= ((uint32_t)c & 0xffu) << (8 * i);
  }
  return w;
}

template <int D, bool IN16, bool OUT16, bool Q8>
__global__ void __launch_bounds__(kAppThreads) norm_rope_append_kernel(const AppendArgs p) {
  constexpr int L = D / 8;                     // lanes per head
  constexpr int kPerCta = kAppThreads / L;     // heads a CTA takes at a time
  griddep_launch();
  griddep_wait();
  const int heads = p.hq + 2 * p.hkv;
  const int64_t units = p.rows * heads, u0 = (int64_t)blockIdx.x * (kPerCta * kUnits) + threadIdx.x / L;
  const int l = threadIdx.x % L, j = 4 * l;
  // every load that depends on the unit's index alone is issued for all of a thread's units before any is used
  float4 a[kUnits], b[kUnits];
  int slot[kUnits], pos[kUnits], hd[kUnits];
  int64_t row[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const int64_t u = u0 + k * kPerCta;
    const bool live = u < units;
    row[k] = live ? (u <= 0x7fffffff ? (int64_t)((uint32_t)u / (uint32_t)heads) : u / heads) : 0;
    hd[k] = live ? (int)(u - row[k] * heads) : 0;
    slot[k] = live ? __ldg(p.slots + row[k]) : -1;
    pos[k] = live && p.cos_sin ? __ldg(p.positions + row[k]) : 0;
    const int64_t at = row[k] * p.ld + (int64_t)hd[k] * D + j;
    if (live) {
      a[k] = load4<IN16>(p.qkv, at);
      b[k] = load4<IN16>(p.qkv, at + D / 2);
    } else {
      a[k] = b[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const bool on = slot[k] >= 0;  // a negative slot: a padding row (or no unit), left as it is
    const bool is_q = hd[k] < p.hq, is_k = !is_q && hd[k] < p.hq + p.hkv;
    const float* w = is_q ? p.qw : (is_k ? p.kw : nullptr);
    float4 x = a[k], y = b[k];
    if (p.qw || p.kw) {  // (uniform: every lane takes part in the shuffles)
      float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (w) {
        const float inv = rsqrtf(ss * (1.f / D) + p.eps);
        const float4 wa = __ldg(reinterpret_cast<const float4*>(w + j)), wb = __ldg(reinterpret_cast<const float4*>(w + D / 2 + j));
        x = make_float4(x.x * inv * wa.x, x.y * inv * wa.y, x.z * inv * wa.z, x.w * inv * wa.w);
        y = make_float4(y.x * inv * wb.x, y.y * inv * wb.y, y.z * inv * wb.z, y.w * inv * wb.w);
      }
    }
    bool ok = on;
    if (p.cos_sin && on) {
      if (pos[k] < 0 || pos[k] >= p.max_pos) {  // (nothing of such a row is written, V neither)
        if (l == 0) mg_record_error(MG_ERR_DEVICE, 210);
        ok = false;
      } else if (is_q || is_k) {
        const float* cs = p.cos_sin + (int64_t)pos[k] * D;
        const float4 c = __ldg(reinterpret_cast<const float4*>(cs + j)), s = __ldg(reinterpret_cast<const float4*>(cs + D / 2 + j));
        const float4 u = x, v = y;
        x = make_float4(u.x * c.x - v.x * s.x, u.y * c.y - v.y * s.y, u.z * c.z - v.z * s.z, u.w * c.w - v.w * s.w);
        y = make_float4(v.x * c.x + u.x * s.x, v.y * c.y + u.y * s.y, v.z * c.z + u.z * s.z, v.w * c.w + u.w * s.w);
      }
    }
    float mx = 0.f;
    if constexpr (Q8) {
      mx = max_nan(max_nan(max_nan(fabsf(x.x), fabsf(x.y)), max_nan(fabsf(x.z), fabsf(x.w))),
                   max_nan(max_nan(fabsf(y.x), fabsf(y.y)), max_nan(fabsf(y.z), fabsf(y.w))));
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (!ok) continue;
    if (is_q) {
      const int64_t at = (row[k] * p.hq + hd[k]) * D + j;
      if constexpr (OUT16) {
        __nv_bfloat16* q = static_cast<__nv_bfloat16*>(p.q_out) + at;
        store4_bf16(q, x);
        store4_bf16(q + D / 2, y);
      } else {
        float* q = static_cast<float*>(p.q_out) + at;
        *reinterpret_cast<float4*>(q) = x;
        *reinterpret_cast<float4*>(q + D / 2) = y;
      }
      continue;
    }
    const int64_t blk = slot[k] >> 4;
    if (blk >= p.num_blocks) {
      if (l == 0) mg_record_error(MG_ERR_DEVICE, 211);
      continue;
    }
    const int kh = hd[k] - p.hq - (is_k ? 0 : p.hkv);
    const int64_t at = (blk * p.hkv + kh) * 16 + (slot[k] & 15);
    if constexpr (Q8) {
      const float s = max_nan(__fdiv_rn(mx, 127.f), 1e-8f);
      uint8_t* dst = static_cast<uint8_t*>(is_k ? p.k_pool : p.v_pool) + at * D + j;
      *reinterpret_cast<uint32_t*>(dst) = code4(x, s);
      *reinterpret_cast<uint32_t*>(dst + D / 2) = code4(y, s);
      if (l == 0) (is_k ? p.k_scales : p.v_scales)[at] = s;
    } else {
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(is_k ? p.k_pool : p.v_pool) + at * D + j;
      store4_bf16(dst, x);
      store4_bf16(dst + D / 2, y);
    }
  }
}

template <int D, bool IN16, bool OUT16>
int launch_append(const AppendArgs& a, bool q8, cudaStream_t st) {
  const int64_t units = a.rows * (a.hq + 2 * a.hkv), per = (int64_t)kAppThreads / (D / 8) * kUnits;
  const int64_t grid = (units + per - 1) / per;
  if (grid > 0x7fffffff) return MG_ERR_UNSUPPORTED;
  if (q8)
    MG_CUDA_TRY(mg_launch(norm_rope_append_kernel<D, IN16, OUT16, true>, dim3((unsigned)grid), dim3(kAppThreads), 0,
                          st, 1, a));
  else
    MG_CUDA_TRY(mg_launch(norm_rope_append_kernel<D, IN16, OUT16, false>, dim3((unsigned)grid), dim3(kAppThreads), 0,
                          st, 1, a));
  MG_LAUNCH_CHECK();
  return MG_OK;
}

template <int D>
int launch_append_types(const AppendArgs& a, bool in16, bool out16, bool q8, cudaStream_t st) {
  if (in16) return out16 ? launch_append<D, true, true>(a, q8, st) : launch_append<D, true, false>(a, q8, st);
  return out16 ? launch_append<D, false, true>(a, q8, st) : launch_append<D, false, false>(a, q8, st);
}

}  // namespace

extern "C" int mg_norm_rope_kv_append(const void* qkv, int qkv_bf16, int64_t ld_qkv, int64_t rows,
                                      const int32_t* positions, const float* cos_sin, int max_pos,
                                      const int32_t* slots, const float* q_weight, const float* k_weight, float eps,
                                      int hq, int hkv, int d, void* q_out, int q_bf16, void* k_pool, void* v_pool,
                                      float* k_scales, float* v_scales, int64_t num_blocks, void* stream) {
  const bool q8 = k_scales != nullptr;
  if (rows < 0 || hq <= 0 || hkv <= 0 || hq % hkv || num_blocks <= 0 || !k_pool || !v_pool || q8 != (v_scales != nullptr) ||
      ld_qkv < (int64_t)(hq + 2 * hkv) * d || ld_qkv % 4 || (rows > 0 && (!qkv || !slots || !q_out)) ||
      (cos_sin && ((rows > 0 && !positions) || max_pos <= 0)))
    return MG_ERR_INVALID_ARG;
  if (d != 32 && d != 64 && d != 128) return MG_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(cos_sin) | reinterpret_cast<uintptr_t>(q_weight) |
       reinterpret_cast<uintptr_t>(k_weight) | reinterpret_cast<uintptr_t>(q_out) |
       reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15)
    return MG_ERR_INVALID_ARG;
  if (rows == 0) return MG_OK;
  // (heads are read and written in any order)
  if (mg_overlap(qkv, ((rows - 1) * ld_qkv + (int64_t)(hq + 2 * hkv) * d) * (qkv_bf16 ? 2 : 4), q_out,
                 rows * hq * d * (q_bf16 ? 2 : 4)))
    return MG_ERR_INVALID_ARG;
  AppendArgs a{};
  a.qkv = qkv;
  a.ld = ld_qkv;
  a.rows = rows;
  a.positions = positions;
  a.slots = slots;
  a.cos_sin = cos_sin;
  a.qw = q_weight;
  a.kw = k_weight;
  a.eps = eps;
  a.max_pos = max_pos;
  a.hq = hq;
  a.hkv = hkv;
  a.q_out = q_out;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.num_blocks = num_blocks;
  cudaStream_t st = mg_stream(stream);
  if (d == 32) return launch_append_types<32>(a, qkv_bf16, q_bf16, q8, st);
  if (d == 64) return launch_append_types<64>(a, qkv_bf16, q_bf16, q8, st);
  return launch_append_types<128>(a, qkv_bf16, q_bf16, q8, st);
}
