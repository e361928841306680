// Verification of drafted tokens against the target's probabilities (the rejection rule of speculative sampling).
// Request i owns logits rows cu[i] .. cu[i+1]-1: row j of it was computed from the tokens up to the j-th draft and
// asks about the next one, d_j = tokens[cu[i] + j + 1]; the last row asks about none. With temperature T > 0,
//   p = softmax(logits / T), q = the draft's distribution (one-hot where none is given),
//   d_j is accepted iff u_j q(d_j) < p(d_j), in order until the first that is not;
//   then a token is drawn from max(p - q, 0) of that row (from p where that is zero everywhere, and of the last
//   row where every draft was accepted): the first index whose running sum passes u_last times the whole.
// T = 0 is greedy: d_j is accepted iff it is the row's first maximal index, and that index is the token.
//
// Two launches. The first streams every row once and leaves (max, sum of exponentials, argmax) per chunk: bound by
// memory. The second, one cluster of CTAs per request, decides from those where the request stops, and works on that
// one row alone. Its sums are in 64 bits: with 10^5 entries the running sum's steps are so close that 32-bit sums
// put the drawn index one off in about one of a hundred draws, where 64-bit sums of 64-bit exponentials do in none.
#include <float.h>

#include "common.cuh"

namespace {

constexpr int kStatThreads = 256;
constexpr int kStatVec = 8;                              // float4 loads in flight per thread
constexpr int kStatChunk = kStatThreads * 4 * kStatVec;  // logits per CTA
constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kPickCtas = 8;
constexpr int kPickBatch = 8;                            // loads in flight per thread
constexpr int kPickStore = 200 * 1024;                   // shared memory for a CTA's share of the weights

struct VerifyArgs {
  const float* logits;
  int64_t ld, ldq;
  const float* probs;
  const int32_t *tokens, *cu;
  const float *uniforms, *temps;
  int64_t vocab;
  int64_t rows;
  int b, chunks;
  float4* stats;  // [rows][chunks]: max, sum exp((x - max) / T), argmax (bits), unused
  int32_t *accepted, *next;
};

// (m, s) <- merge of two (max, sum of exp2((x - max) * c)) states.
__device__ __forceinline__ void merge_ms(float& m, float& s, float om, float os, float c) {
  const float nm = fmaxf(m, om);
  s = (m == -INFINITY ? 0.f : s * exp2f((m - nm) * c)) + (om == -INFINITY ? 0.f : os * exp2f((om - nm) * c));
  m = nm;
}

__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const VerifyArgs p) {
  griddep_launch();
  griddep_wait();
  __shared__ float sm_m[kStatThreads / 32], sm_s[kStatThreads / 32], sm_v[kStatThreads / 32];
  __shared__ int32_t sm_i[kStatThreads / 32];
  const int64_t row = blockIdx.y;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const float* x = p.logits + row * p.ld;
  const int64_t lo = (int64_t)blockIdx.x * kStatChunk, hi = min(lo + (int64_t)kStatChunk, p.vocab);
  float v[4 * kStatVec];
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
#pragma unroll
  for (int k = 0; k < kStatVec; ++k) {
    const int64_t i = lo + 4 * ((int64_t)k * kStatThreads + t);
    if (vec && i + 4 <= hi) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(x + i));
      v[4 * k] = f.x, v[4 * k + 1] = f.y, v[4 * k + 2] = f.z, v[4 * k + 3] = f.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * k + e] = i + e < hi ? x[i + e] : -INFINITY;
    }
  }
  // (while the loads are under way) the request that owns the row: the starts at or before it, less one
  int seen = 0;
  for (int i0 = 0; i0 <= p.b; i0 += kStatThreads)
    seen += __syncthreads_count(i0 + t <= p.b && p.cu[i0 + t] <= row);
  const int req = seen - 1;
  if (req < 0 || req >= p.b) return;  // a row behind the last request
  const float T = p.temps ? p.temps[req] : 1.f;
  const float c = T > 0.f ? 1.4426950408889634f / T : 0.f;
  float m = -INFINITY, s = 0.f, best = -INFINITY;
  int32_t bi = 0x7fffffff;
  if (T > 0.f) {
    bool nan = false;
#pragma unroll
    for (int k = 0; k < 4 * kStatVec; ++k) {
      m = fmaxf(m, v[k]);
      nan |= v[k] != v[k];
    }
    if (m != -INFINITY) {
#pragma unroll
      for (int k = 0; k < 4 * kStatVec; ++k) s += exp2f((v[k] - m) * c);
    }
    if (nan) s = NAN;
    if (m == -INFINITY && nan) m = 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      merge_ms(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o), c);
  } else {
#pragma unroll
    for (int k = 0; k < kStatVec; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t i = lo + 4 * ((int64_t)k * kStatThreads + t) + e;
        if (i < hi && mg_argmax_better(v[4 * k + e], (int32_t)i, best, bi)) {
          best = v[4 * k + e];
          bi = (int32_t)i;
        }
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, best, o);
      const int32_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (mg_argmax_better(ov, oi, best, bi)) {
        best = ov;
        bi = oi;
      }
    }
  }
  if (lane == 0) {
    sm_m[w] = m;
    sm_s[w] = s;
    sm_v[w] = best;
    sm_i[w] = bi;
  }
  __syncthreads();
  if (t == 0) {
    for (int k = 1; k < kStatThreads / 32; ++k) {
      if (T > 0.f) {
        merge_ms(m, s, sm_m[k], sm_s[k], c);
      } else if (mg_argmax_better(sm_v[k], sm_i[k], best, bi)) {
        best = sm_v[k];
        bi = sm_i[k];
      }
    }
    p.stats[row * p.chunks + blockIdx.x] = make_float4(T > 0.f ? m : best, s, __int_as_float(bi), 0.f);
  }
}

// The state of a row from its chunks, by one warp: (m, s) of the softmax, or (greedy) the first maximal index.
__device__ __forceinline__ void row_state(const float4* st, int chunks, int lane, bool greedy, float c, float& m,
                                          float& s, int32_t& bi) {
  float best = -INFINITY;
  m = -INFINITY;
  s = 0.f;
  bi = 0x7fffffff;
  auto take = [&](float v, int32_t i) {
    if (mg_argmax_better(v, i, best, bi)) {
      best = v;
      bi = i;
    }
  };
  for (int k = lane; k < chunks; k += 32) {
    const float4 v = st[k];
    if (greedy) take(v.x, __float_as_int(v.z)); else merge_ms(m, s, v.x, v.y, c);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (greedy) {
      const float ov = __shfl_xor_sync(0xffffffffu, best, o);
      const int32_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
      take(ov, oi);
    } else {
      const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
      merge_ms(m, s, om, os, c);
    }
  }
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double ld_dsmem_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr));
  return v;
}

// Sum over the cluster's CTAs and warps of each warp's `mine`, and (before) the sum of those before this warp, in
// (CTA, warp) order. part: kPickWarps doubles of shared memory, free for reuse after the next cluster barrier.
__device__ __forceinline__ double cluster_total(double mine, double* part, int w, int lane, double* before) {
  if (lane == 0) part[w] = mine;
  cluster_sync_all();
  const uint32_t rank = cluster_ctarank();
  double total = 0.0, pre = 0.0;
#pragma unroll
  for (int k = lane; k < kPickCtas * kPickWarps; k += 32) {
    const uint32_t r = (uint32_t)(k / kPickWarps);
    const double v = ld_dsmem_f64(mapa_shared(smem_u32(part + k % kPickWarps), r));
    total += v;
    if ((int)r < (int)rank || (r == rank && k % kPickWarps < w)) pre += v;
  }
  if (before) *before = warp_sum_d(pre);
  return warp_sum_d(total);
}

template <bool kStored>
__global__ void __launch_bounds__(kPickThreads) verify_pick_kernel(const VerifyArgs p) {
  extern __shared__ double weights[];
  griddep_launch();
  griddep_wait();
  __shared__ int s_stop, s_bad;
  __shared__ double part_z[kPickWarps], part_r[kPickWarps], part_p[kPickWarps];
  __shared__ float s_max;
  __shared__ int s_found;
  const int req = (int)blockIdx.y, rank = (int)blockIdx.x;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int64_t r0 = p.cu[req], r1 = p.cu[req + 1];
  if (r0 < 0 || r1 > p.rows || r1 <= r0) {  // no rows: nothing to ask (the whole cluster leaves together)
    if (rank == 0 && t == 0) {
      if (r0 != r1) mg_record_error(MG_ERR_DEVICE, 601);
      p.accepted[req] = 0;
      p.next[req] = -1;
    }
    return;
  }
  const int n = (int)(r1 - r0 - 1);
  const float T = p.temps ? p.temps[req] : 1.f;
  const bool greedy = !(T > 0.f);
  const float c = greedy ? 0.f : 1.4426950408889634f / T;
  if (t == 0) {
    s_stop = n;
    s_bad = T < 0.f || T != T ? 602 : 0;
    s_found = 0x7fffffff;
  }
  __syncthreads();
  // one warp per row: the row's state from its chunks, then the test of its draft
  for (int j = w; j <= n; j += kPickWarps) {
    float m, sum;
    int32_t bi;
    row_state(p.stats + (r0 + j) * p.chunks, p.chunks, lane, greedy, c, m, sum, bi);
    if (lane == 0) {
      bool ok = false;
      if (j < n) {
        const int32_t d = p.tokens[r0 + j + 1];
        if (d < 0 || d >= p.vocab) {
          atomicMax(&s_bad, 603);
        } else if (greedy) {
          ok = d == bi;
        } else {
          const double pd = exp(((double)p.logits[(r0 + j) * p.ld + d] - (double)m) / (double)T) / (double)sum;
          const double qd = p.probs ? (double)p.probs[(r0 + j) * p.ldq + d] : 1.0;
          ok = (double)p.uniforms[r0 + j] * qd < pd;
        }
      }
      if (!ok) atomicMin(&s_stop, j);
    }
  }
  __syncthreads();
  const int stop = s_stop;
  if (w == 0) {  // the stopping row's state again (its warp did not know that it would be the one)
    float m, sum;
    int32_t bi;
    row_state(p.stats + (r0 + stop) * p.chunks, p.chunks, lane, greedy, c, m, sum, bi);
    if (lane == 0) {
      s_max = m;
      if (!greedy && (m == -INFINITY || m == INFINITY || sum != sum)) atomicMax(&s_bad, 604);
      if (greedy) s_found = bi == 0x7fffffff ? 0 : bi;
    }
  }
  __syncthreads();
  const int bad = s_bad;
  if (bad && rank == 0 && t == 0) mg_record_error(MG_ERR_DEVICE, bad);
  // (every CTA of the cluster has taken the same decisions from the same data)
  if (greedy || bad == 602 || bad == 604) {
    if (rank == 0 && t == 0) {
      p.accepted[req] = bad == 602 ? 0 : stop;
      p.next[req] = bad == 602 || bad == 604 ? -1 : s_found;
    }
    return;
  }

  // ---- draw from the stopping row ----
  const float* x = p.logits + (r0 + stop) * p.ld;
  const float* qrow = stop < n && p.probs ? p.probs + (r0 + stop) * p.ldq : nullptr;
  const int64_t hole = stop < n && !p.probs ? (int64_t)p.tokens[r0 + stop + 1] : -1;  // a one-hot draft's token
  const double mx = (double)s_max, inv_t = 1.0 / (double)T;
  // each warp owns a contiguous run of the vocabulary; in the stored form its weights stay in shared memory
  const int64_t nw = kPickCtas * kPickWarps, run = (p.vocab + nw - 1) / nw;
  const int64_t me = (int64_t)rank * kPickWarps + w;
  const int64_t v0 = min(me * run, p.vocab);
  const int len = (int)(min(v0 + run, p.vocab) - v0);
  double* kept = weights + (kStored ? (int64_t)w * run : 0);
  auto weight = [&](int64_t v) -> double { return exp(((double)x[v] - mx) * inv_t); };
  double z = 0.0, holed = 0.0;
  for (int i0 = lane; i0 < len; i0 += 32 * kPickBatch) {
    float l[kPickBatch];
#pragma unroll
    for (int k = 0; k < kPickBatch; ++k) l[k] = i0 + 32 * k < len ? __ldg(x + v0 + i0 + 32 * k) : 0.f;
#pragma unroll
    for (int k = 0; k < kPickBatch; ++k) {
      const int i = i0 + 32 * k;
      if (i < len) {
        double e = exp(((double)l[k] - mx) * inv_t);
        z += e;
        if (v0 + i == hole) e = 0.0;  // nothing is left of it
        holed += e;
        if (kStored) kept[i] = e;
      }
    }
  }
  z = warp_sum_d(z);
  const double Z = cluster_total(z, part_z, w, lane, nullptr), inv_z = 1.0 / Z;
  bool plain = stop >= n;  // the draw is from p itself
  double mine = warp_sum_d(holed);
  if (qrow) {
    mine = 0.0;
    for (int i0 = lane; i0 < len; i0 += 32 * kPickBatch) {
      float q[kPickBatch];
#pragma unroll
      for (int k = 0; k < kPickBatch; ++k) q[k] = i0 + 32 * k < len ? __ldg(qrow + v0 + i0 + 32 * k) : 0.f;
#pragma unroll
      for (int k = 0; k < kPickBatch; ++k) {
        const int i = i0 + 32 * k;
        if (i < len) {
          const double e = kStored ? kept[i] : weight(v0 + i), rest = fmax(e * inv_z - (double)q[k], 0.0);
          mine += rest;
          if (kStored) kept[i] = rest;
        }
      }
    }
    mine = warp_sum_d(mine);
  }
  double before, total = cluster_total(mine, part_r, w, lane, &before);
  if (!plain && !(total > 0.0)) {  // p and q alike in every place: the draw is from p
    plain = true;
    total = cluster_total(z, part_p, w, lane, &before);
    mine = z;
    if (kStored)
      for (int i = lane; i < len; i += 32) kept[i] = weight(v0 + i);
  }
  auto rest_at = [&](int i) -> double {
    if (kStored) return kept[i];
    if (plain) return weight(v0 + i);
    if (v0 + i == hole) return 0.0;
    const double e = weight(v0 + i);
    return qrow ? fmax(e * inv_z - (double)qrow[v0 + i], 0.0) : e;
  };
  const double target = (double)p.uniforms[r1 - 1] * total;
  // the first index whose running sum passes the target: in one warp's run, a contiguous piece of it for each lane
  if (before <= target && before + mine > target) {
    __syncwarp();
    const int piece = ((len + 31) / 32) | 1;  // (odd: the lanes' pieces start in different banks)
    const int a = min(lane * piece, len), e = min(a + piece, len);
    double sum = 0.0;
    int last = -1;
    for (int i = a; i < e; ++i) {
      const double v = rest_at(i);
      sum += v;
      if (v > 0.0) last = i;
    }
    double cum = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, cum, o);
      if (lane >= o) cum += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, last >= 0 && before + cum > target);
    const unsigned any = __ballot_sync(0xffffffffu, last >= 0);
    // (where the sums' last bits leave no lane: the last index with any weight)
    const int take = hit ? __ffs(hit) - 1 : (any ? 31 - __clz(any) : -1);
    if (lane == take) {
      double at = before + cum - sum;
      int found = last;
      for (int i = a; i < e; ++i) {
        const double v = rest_at(i);
        at += v;
        if (v > 0.0 && at > target) {
          found = i;
          break;
        }
      }
      atomicMin(&s_found, (int)(v0 + found));
    }
  }
  cluster_sync_all();
  if (rank == 0 && w == 0) {
    int best = 0x7fffffff;
    if (lane < kPickCtas) {
      uint32_t v;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(&s_found), (uint32_t)lane)));
      best = (int)v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (best == 0x7fffffff) {  // only rounding leaves none: the last index with any weight
      for (int64_t g = (p.vocab + 31) / 32 - 1; g >= 0 && best == 0x7fffffff; --g) {
        const int64_t v = g * 32 + lane;
        double rest = 0.0;
        if (v < p.vocab && v != (plain ? -1 : hole)) {
          rest = weight(v);
          if (!plain && qrow) rest = fmax(rest * inv_z - (double)qrow[v], 0.0);
        }
        const unsigned any = __ballot_sync(0xffffffffu, rest > 0.0);
        if (any) best = (int)(g * 32) + 31 - __clz(any);
      }
    }
    if (lane == 0) {
      p.accepted[req] = stop;
      p.next[req] = best == 0x7fffffff ? -1 : best;
    }
  }
  cluster_sync_all();  // the other CTAs' results stay readable until rank 0 has read them
}

}  // namespace

extern "C" int mg_verify_workspace_bytes(int64_t rows, int64_t vocab, size_t* bytes) {
  if (!bytes || rows < 0 || vocab <= 0) return MG_ERR_INVALID_ARG;
  if (vocab > 0x7fffffc0 || rows > 65535) return MG_ERR_UNSUPPORTED;
  *bytes = (size_t)rows * (size_t)((vocab + kStatChunk - 1) / kStatChunk) * sizeof(float4);
  return MG_OK;
}

extern "C" int mg_verify_drafts(const float* logits, int64_t ld, int64_t rows, int64_t vocab, const int32_t* tokens,
                                const int32_t* cu_rows, int b, const float* draft_probs, int64_t ld_probs,
                                const float* uniforms, const float* temperatures, int32_t* accepted, int32_t* next,
                                void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  const int rc = mg_verify_workspace_bytes(rows, vocab, &need);
  if (rc) return rc;
  if (b < 0 || ld < vocab || (draft_probs && ld_probs < vocab) ||
      (b > 0 && (!cu_rows || !accepted || !next)) || (rows > 0 && (!logits || !tokens || !uniforms)) ||
      workspace_bytes < need || (need && !workspace) || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return MG_ERR_INVALID_ARG;
  if (b > 65535) return MG_ERR_UNSUPPORTED;
  if (b == 0) return MG_OK;
  VerifyArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.probs = draft_probs;
  a.ldq = ld_probs;
  a.tokens = tokens;
  a.cu = cu_rows;
  a.uniforms = uniforms;
  a.temps = temperatures;
  a.vocab = vocab;
  a.rows = rows;
  a.b = b;
  a.chunks = (int)((vocab + kStatChunk - 1) / kStatChunk);
  a.stats = static_cast<float4*>(workspace);
  a.accepted = accepted;
  a.next = next;
  cudaStream_t st = mg_stream(stream);
  if (rows > 0)
    MG_CUDA_TRY(mg_launch(verify_stats_kernel, dim3((unsigned)a.chunks, (unsigned)rows), dim3(kStatThreads), 0, st, 1, a));
  // The row's weights are kept in shared memory between the passes while a CTA's eighth of them fits (vocabularies to
  // 204800); beyond that they are computed again in each.
  const int64_t nw = kPickCtas * kPickWarps, kept = (vocab + nw - 1) / nw * kPickWarps * (int64_t)sizeof(double);
  if (kept <= kPickStore) {
    static bool done[64] = {};
    static std::mutex mu;
    MG_CUDA_TRY(mg_once_per_device(done, mu, [] {
      return cudaFuncSetAttribute(verify_pick_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPickStore);
    }));
    MG_CUDA_TRY(mg_launch(verify_pick_kernel<true>, dim3(kPickCtas, (unsigned)b), dim3(kPickThreads), (size_t)kept, st,
                          kPickCtas, a));
  } else {
    MG_CUDA_TRY(mg_launch(verify_pick_kernel<false>, dim3(kPickCtas, (unsigned)b), dim3(kPickThreads), 0, st, kPickCtas, a));
  }
  MG_LAUNCH_CHECK();
  return MG_OK;
}
