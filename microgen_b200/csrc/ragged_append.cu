// Norms of queries and keys for each head, rotary positions, and the paged K/V append, in one pass over the QKV
// projection's rows. For a head vector x of d values at position p:
//   y = x * rsqrt(mean(x^2) + eps) * w          (q and k heads, where a weight is given)
//   z_j = y_j cos_j - y_{j+d/2} sin_j,  z_{j+d/2} = y_{j+d/2} cos_j + y_j sin_j   (q and k heads, where a table is)
// q goes out in bf16 or fp32, K and V into their slot of the pools in bf16, or as int8 codes with one scale per
// vector: s = max(max|z| / 127, 1e-8), code = clamp(round_half_even(z / s), -128, 127).
//
// Bound by memory: every value is read once and written once. d / 8 lanes hold a head, each with four adjacent
// values of the first half and their four rotation partners of the second, so that loads are 16 bytes, the
// rotation needs no exchange, and a norm or an absolute maximum is a few shuffles. All sums are fp32; the one
// rounding is the store (q and K/V feed bf16 tensor-core products).
#include "common.cuh"

namespace {

constexpr int kAppThreads = 256;

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

__device__ __forceinline__ uint32_t code4(const float4& a, float s) {
  const float v[4] = {a.x, a.y, a.z, a.w};
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = fminf(fmaxf(rintf(__fdiv_rn(v[i], s)), -128.f), 127.f);
    w |= ((uint32_t)(int)c & 0xffu) << (8 * i);
  }
  return w;
}

template <int D, bool IN16, bool OUT16, bool Q8>
__global__ void __launch_bounds__(kAppThreads) norm_rope_append_kernel(const AppendArgs p) {
  constexpr int L = D / 8;  // lanes per head
  griddep_launch();
  griddep_wait();
  const int heads = p.hq + 2 * p.hkv;
  const int64_t units = p.rows * heads;
  const int64_t u = ((int64_t)blockIdx.x * kAppThreads + threadIdx.x) / L;
  const int l = threadIdx.x % L;
  const bool live = u < units;
  const int64_t r = live ? u / heads : 0;
  const int hd = live ? (int)(u - r * heads) : 0;
  const int slot = live ? p.slots[r] : -1;
  const bool on = live && slot >= 0;  // slot -1: a padding row, left as it is
  const int j = 4 * l;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
  if (on) {
    const int64_t at = r * p.ld + (int64_t)hd * D + j;
    a = load4<IN16>(p.qkv, at);
    b = load4<IN16>(p.qkv, at + D / 2);
  }
  const bool is_q = hd < p.hq, is_k = !is_q && hd < p.hq + p.hkv;
  const float* w = is_q ? p.qw : (is_k ? p.kw : nullptr);
  if (p.qw || p.kw) {  // (uniform: every lane takes part in the shuffles)
    float ss = a.x * a.x + a.y * a.y + a.z * a.z + a.w * a.w + b.x * b.x + b.y * b.y + b.z * b.z + b.w * b.w;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w) {
      const float inv = rsqrtf(ss * (1.f / D) + p.eps);
      const float4 wa = *reinterpret_cast<const float4*>(w + j), wb = *reinterpret_cast<const float4*>(w + D / 2 + j);
      a = make_float4(a.x * inv * wa.x, a.y * inv * wa.y, a.z * inv * wa.z, a.w * inv * wa.w);
      b = make_float4(b.x * inv * wb.x, b.y * inv * wb.y, b.z * inv * wb.z, b.w * inv * wb.w);
    }
  }
  bool ok = on;
  if (p.cos_sin && on && (is_q || is_k)) {
    const int pos = p.positions[r];
    if (pos < 0 || pos >= p.max_pos) {
      if (l == 0) mg_record_error(MG_ERR_DEVICE, 210);
      ok = false;
    } else {
      const float* cs = p.cos_sin + (int64_t)pos * D;
      const float4 c = *reinterpret_cast<const float4*>(cs + j), s = *reinterpret_cast<const float4*>(cs + D / 2 + j);
      const float4 x = a, y = b;
      a = make_float4(x.x * c.x - y.x * s.x, x.y * c.y - y.y * s.y, x.z * c.z - y.z * s.z, x.w * c.w - y.w * s.w);
      b = make_float4(y.x * c.x + x.x * s.x, y.y * c.y + x.y * s.y, y.z * c.z + x.z * s.z, y.w * c.w + x.w * s.w);
    }
  }
  float mx = 0.f;
  if constexpr (Q8) {
    mx = fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))),
               fmaxf(fmaxf(fabsf(b.x), fabsf(b.y)), fmaxf(fabsf(b.z), fabsf(b.w))));
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (!ok) return;
  if (is_q) {
    const int64_t at = (r * p.hq + hd) * D + j;
    if constexpr (OUT16) {
      __nv_bfloat16* q = static_cast<__nv_bfloat16*>(p.q_out) + at;
      store4_bf16(q, a);
      store4_bf16(q + D / 2, b);
    } else {
      float* q = static_cast<float*>(p.q_out) + at;
      *reinterpret_cast<float4*>(q) = a;
      *reinterpret_cast<float4*>(q + D / 2) = b;
    }
    return;
  }
  const int64_t blk = slot >> 4;
  if (blk >= p.num_blocks) {
    if (l == 0) mg_record_error(MG_ERR_DEVICE, 211);
    return;
  }
  const int kh = hd - p.hq - (is_k ? 0 : p.hkv);
  const int64_t row = (blk * p.hkv + kh) * 16 + (slot & 15);
  if constexpr (Q8) {
    const float s = fmaxf(__fdiv_rn(mx, 127.f), 1e-8f);
    uint8_t* dst = static_cast<uint8_t*>(is_k ? p.k_pool : p.v_pool) + row * D + j;
    *reinterpret_cast<uint32_t*>(dst) = code4(a, s);
    *reinterpret_cast<uint32_t*>(dst + D / 2) = code4(b, s);
    if (l == 0) (is_k ? p.k_scales : p.v_scales)[row] = s;
  } else {
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(is_k ? p.k_pool : p.v_pool) + row * D + j;
    store4_bf16(dst, a);
    store4_bf16(dst + D / 2, b);
  }
}

template <int D, bool IN16, bool OUT16>
int launch_append(const AppendArgs& a, bool q8, cudaStream_t st) {
  const int64_t units = a.rows * (a.hq + 2 * a.hkv);
  const int64_t grid = (units * (D / 8) + kAppThreads - 1) / kAppThreads;
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
