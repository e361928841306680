// Verification of drafted tokens against the target's probabilities (the rejection rule of speculative sampling).
// Request i owns logits rows cu[i] .. cu[i+1]-1: row j of it was computed from the tokens up to the j-th draft and
// asks about the next one, d_j = tokens[cu[i] + j + 1]; the last row asks about none. With temperature T > 0,
//   p = softmax(logits / T), q = the draft's distribution (one-hot where none is given),
//   d_j is accepted iff u_j q(d_j) < p(d_j), in order until the first that is not;
//   then a token is drawn from max(p - q, 0) of that row (from p where that is zero everywhere, and of the last
//   row where every draft was accepted): the first index whose running sum passes u_last times the whole.
// T = 0 is greedy: d_j is accepted iff it is the row's first maximal index, and that index is the token.
//
// Every row is streamed once by the first launch, which leaves (max, sum of exponentials, argmax) per chunk: bound by
// memory. The others work on one row per request: they decide from those states where it stops and sum the stopping
// row's weights by segments (decide), and the sums of max(p - q, 0) where the draft has probabilities (rest); the CTA that
// sums a request's last segment finds the index in the segment that the target falls into. Small grids that fill the
// machine measured less (84 us against 103, for 48 requests) than one cluster per request holding the row's weights in
// shared memory, whose eight CTAs of 128 KB find room a third at a time. The draw's sums are in 64 bits: with 10^5 entries
// the running sum's steps are so close that 32-bit sums put the drawn index one off in about one of a hundred draws,
// where 64-bit sums of 64-bit exponentials do in none.
// The test of a draft holds p(d) against the 32-bit sum of the row's state: approximate exponentials of arguments up to 20
// or so that matter (2^-18.5 relative at the most, three roundings of the argument) and a sum of 32 terms a thread, then of
// threads and chunks (2^-19). A draft whose u q(d) lies closer to p(d) than 2^-17 of it may fall either way: at most one of
// 65 thousand drafts.
// 48 requests of 1 to 8 drafts, 128256 entries, draft probabilities (162 MB, 25 us at 6.55 TB/s): 82 us. By
// themselves the rows' states take 34, the decision 34 and the rest 31 (they overlap in part): the latter two issue in half of
// their cycles, with the 64-bit pipe at a quarter of its rate and the memory at a tenth: 64-bit exponentials, each a long chain
// of instructions, on every entry of the stopping row. One request of 4 drafts, 50257 entries: 17 us, of which the decision is
// 15 on 16 CTAs: barriers and dependent loads, each CTA reading all of the request's states before its segment.
#include "common.cuh"

namespace {

constexpr int kStatThreads = 256;
constexpr int kStatVec = 8;                              // float4 loads in flight per thread
constexpr int kStatChunk = kStatThreads * 4 * kStatVec;  // logits per CTA
constexpr int kPickBatch = 8;                            // loads in flight per thread
constexpr int kSegments = 16;                            // of the stopping row, one per CTA
constexpr int kRuns = kSegments * (kStatThreads / 32);   // of the stopping row, one per warp

struct Decision;

struct VerifyArgs {
  const float* logits;
  int64_t ld, ldq;
  const float* probs;
  const int32_t *tokens, *cu;
  const float *uniforms, *temps;
  int64_t vocab;
  int64_t rows;
  int b, chunks;
  float4* stats;        // [rows][chunks]: max, sum exp((x - max) / T), argmax (bits), unused
  Decision* decisions;  // [b]
  double2* parts;       // [b][runs]: sum of the weights, and of those the one-hot draft leaves
  double* rest;         // [b][runs]: sum of max(p - q, 0)
  int32_t* counters;    // [b][2]: segments summed, in the decision and in the rest
  int32_t *accepted, *next;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log2(e) / T, finite for the smallest T too: the maximum's own exponent is 0 times it.
__device__ __forceinline__ float exponent_factor(float T) {
  return T > 0.f ? fminf(1.4426950408889634f / T, 3.402823466e38f) : 0.f;
}

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
  if (blockIdx.x == 0 && row == 0)
    for (int i = t; i < 2 * p.b; i += kStatThreads) p.counters[i] = 0;
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
  const float c = exponent_factor(T);
  float m = -INFINITY, s = 0.f, best = -INFINITY;
  int32_t bi = 0x7fffffff;
  if (T > 0.f) {
    // the chunk's maximum first: exponentials against it need no rescaling when their sums are joined
    bool nan = false;
#pragma unroll
    for (int k = 0; k < 4 * kStatVec; ++k) {
      m = fmaxf(m, v[k]);
      nan |= v[k] != v[k];
    }
    m = warp_max(m);
    if (lane == 0) sm_m[w] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStatThreads / 32; ++k) m = fmaxf(m, sm_m[k]);
    if (m != -INFINITY) {  // (an infinite maximum leaves inf - inf, the NaN that marks the row)
#pragma unroll
      for (int k = 0; k < 4 * kStatVec; ++k) s += ex2((v[k] - m) * c);
    }
    if (nan) s = NAN;
    s = warp_sum(s);
    if (m == -INFINITY && __syncthreads_or(nan)) m = 0.f;
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
    sm_s[w] = s;
    sm_v[w] = best;
    sm_i[w] = bi;
  }
  __syncthreads();
  if (t == 0) {
    for (int k = 1; k < kStatThreads / 32; ++k) {
      if (T > 0.f) {
        s += sm_s[k];
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
// What the decision leaves for the draw.
struct __align__(16) Decision {
  int32_t stop, draw;  // rows kept; 0: answered already, 1: draw from p, 2: draw from what the draft leaves of p
  float max;           // the stopping row's maximum
  int32_t pad;
};

// The stopping row's weights: exp((x - max) / T), and of those max(weight / Z - q, 0) or all but the one-hot draft's.
struct Row {
  const float *x, *q;
  double mx, inv_t, inv_z;
  int64_t hole;
  __device__ __forceinline__ double weight(float l) const { return exp(((double)l - mx) * inv_t); }
  __device__ __forceinline__ double rest(int64_t v) const {
    const double e = v == hole ? 0.0 : weight(__ldg(x + v));
    return q ? fmax(e * inv_z - (double)__ldg(q + v), 0.0) : e;
  }
};
__device__ __forceinline__ Row stopping_row(const VerifyArgs& p, const Decision& d, int req, bool rest) {
  const int64_t r = p.cu[req] + d.stop;
  Row w;
  w.x = p.logits + r * p.ld;
  w.q = rest && p.probs ? p.probs + r * p.ldq : nullptr;
  w.hole = rest && !p.probs ? (int64_t)p.tokens[r + 1] : -1;
  w.mx = (double)d.max;
  w.inv_t = 1.0 / (p.temps ? (double)p.temps[req] : 1.0);
  w.inv_z = 0.0;
  return w;
}

// Run `k` of the vocabulary: [v0, v1).
__device__ __forceinline__ void run_of(int64_t vocab, int k, int64_t& v0, int64_t& v1) {
  const int64_t len = (vocab + kRuns - 1) / kRuns;
  v0 = min((int64_t)k * len, vocab);
  v1 = min(v0 + len, vocab);
}

// Inclusive prefix sum of one double per thread over the CTA; red: a double per warp.
__device__ __forceinline__ double block_prefix(double v, double* red) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) red[w] = v;
  __syncthreads();
  for (int k = 0; k < w; ++k) v += red[k];
  return v;
}

// The draw, by the CTA that sums a request's last segment: the run in which the running sum passes the target, then the
// index within it, a few entries for each thread.
__device__ __forceinline__ void draw_index(const VerifyArgs& p, int req, const Decision& d) {
  static_assert(kRuns <= kStatThreads, "a thread for each run");
  constexpr int kWarps = kStatThreads / 32;
  __shared__ double s_red[2][kWarps], s_total, s_before;
  __shared__ int s_first[2], s_last[2];
  const int t = threadIdx.x;
  if (t < 2) {
    s_first[t] = 0x7fffffff;
    s_last[t] = -1;
  }
  const double2 z = t < kRuns ? __ldcg(p.parts + (int64_t)req * kRuns + t) : make_double2(0.0, 0.0);
  bool rest = d.draw == 2;
  double part = !rest ? z.x : (p.probs ? (t < kRuns ? __ldcg(p.rest + (int64_t)req * kRuns + t) : 0.0) : z.y);
  if (rest && !__syncthreads_or(part > 0.0)) {  // p and q alike in every place: the draw is from p
    rest = false;
    part = z.x;
  }
  double Z = z.x;
  if (rest && p.probs) {  // (the whole of the weights, for p itself)
    Z = block_prefix(z.x, s_red[0]);
    if (t == kStatThreads - 1) s_total = Z;
    __syncthreads();
    Z = s_total;
    __syncthreads();
  }
  const double cum = block_prefix(part, s_red[1]);
  if (t == kStatThreads - 1) s_total = cum;
  __syncthreads();
  const double target = (double)p.uniforms[p.cu[req + 1] - 1] * s_total;
  if (part > 0.0) {
    atomicMax(&s_last[0], t);
    if (cum > target) atomicMin(&s_first[0], t);
  }
  __syncthreads();
  const int run = s_first[0] != 0x7fffffff ? s_first[0] : s_last[0];  // (the last where the sums' last bits leave none)
  if (t == run) s_before = cum - part;
  if (run < 0) {
    if (t == 0) p.next[req] = -1;
    return;
  }
  Row row = stopping_row(p, d, req, rest);
  row.inv_z = 1.0 / Z;
  int64_t v0, v1;
  run_of(p.vocab, run, v0, v1);
  const int64_t piece = (v1 - v0 + kStatThreads - 1) / kStatThreads, a = min(v0 + t * piece, v1), e = min(a + piece, v1);
  double sum = 0.0;
  int64_t last = -1;
#pragma unroll 4
  for (int64_t v = a; v < e; ++v) {
    const double r = row.rest(v);
    sum += r;
    if (r > 0.0) last = v;
  }
  const double in = block_prefix(sum, s_red[0]), base = s_before + (in - sum);  // (its barrier covers s_before)
  if (last >= 0) {
    atomicMax(&s_last[1], t);
    if (base + sum > target) atomicMin(&s_first[1], t);
  }
  __syncthreads();
  const int owner = s_first[1] != 0x7fffffff ? s_first[1] : s_last[1];
  if (t == owner) {
    double at = base;
    int64_t found = last;
    for (int64_t v = a; v < e; ++v) {
      const double r = row.rest(v);
      at += r;
      if (r > 0.0 && at > target) {
        found = v;
        break;
      }
    }
    p.next[req] = (int32_t)found;
  }
  if (owner < 0 && t == 0) p.next[req] = -1;
}

// Whether this CTA's segment is the request's last to be summed (its warps have written their sums, each with a fence).
__device__ __forceinline__ bool last_segment(int32_t* counter) {
  __shared__ int s_done;
  __syncthreads();
  if (threadIdx.x == 0) {
    s_done = atomicAdd(counter, 1) == kSegments - 1;
    __threadfence();
  }
  __syncthreads();
  return s_done != 0;
}

// Decides where request blockIdx.y stops (every CTA for itself, from the rows' states), answers it where no draw is
// needed, and sums one segment of the stopping row: part[0] its weights, part[1] those but the one-hot draft's.
__global__ void __launch_bounds__(kStatThreads) verify_decide_kernel(const VerifyArgs p) {
  griddep_launch();
  griddep_wait();
  constexpr int kWarps = kStatThreads / 32;
  __shared__ int s_stop, s_bad, s_next;
  __shared__ float s_max;
  const int req = (int)blockIdx.y, seg = (int)blockIdx.x;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  Decision* out = p.decisions + req;
  const int64_t r0 = p.cu[req], r1 = p.cu[req + 1];
  if (r0 < 0 || r1 > p.rows || r1 <= r0) {  // no rows: nothing to ask
    if (seg == 0 && t == 0) {
      if (r0 != r1) mg_record_error(MG_ERR_DEVICE, 601);
      p.accepted[req] = 0;
      p.next[req] = -1;
      out->draw = 0;
    }
    return;
  }
  const int n = (int)(r1 - r0 - 1);
  const float T = p.temps ? p.temps[req] : 1.f;
  const bool greedy = !(T > 0.f), bad_t = !(T >= 0.f);
  const float c = exponent_factor(T);
  if (t == 0) {
    s_stop = n;
    s_bad = 0;
  }
  __syncthreads();
  // one warp per row: the row's state from its chunks, then the test of its draft
  for (int j = w; j <= n; j += kWarps) {
    float m, sum;
    int32_t bi, d = -1;
    float ld = 0.f, qd = 1.f, ud = 0.f;
    if (j < n && lane == 0) {  // (under way while the chunks are read)
      d = p.tokens[r0 + j + 1];
      if (d >= 0 && d < p.vocab) {
        ld = p.logits[(r0 + j) * p.ld + d];
        if (p.probs) qd = p.probs[(r0 + j) * p.ldq + d];
      }
      ud = p.uniforms[r0 + j];
    }
    row_state(p.stats + (r0 + j) * p.chunks, p.chunks, lane, greedy, c, m, sum, bi);
    if (lane == 0) {
      bool ok = false;
      if (j < n) {
        if (d < 0 || d >= p.vocab) atomicMax(&s_bad, 603);
        else if (greedy) ok = d == bi;
        else ok = (double)ud * (double)qd < exp(((double)ld - (double)m) / (double)T) / (double)sum;
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
      s_next = bi == 0x7fffffff ? 0 : bi;
      if (!greedy && (m == -INFINITY || m == INFINITY || sum != sum)) atomicMax(&s_bad, 604);
    }
  }
  __syncthreads();
  const int bad = bad_t ? 602 : s_bad;  // (without a temperature there is no answer, whatever else is wrong)
  const bool answered = greedy || bad == 604;
  if (seg == 0 && t == 0) {
    if (bad) mg_record_error(MG_ERR_DEVICE, bad);
    p.accepted[req] = bad_t ? 0 : stop;
    if (answered) p.next[req] = bad_t || bad == 604 ? -1 : s_next;
    out->stop = stop;
    out->max = s_max;
    out->draw = answered ? 0 : (stop < n ? 2 : 1);
  }
  if (answered) return;
  Decision d;
  d.stop = stop;
  d.draw = stop < n ? 2 : 1;
  d.max = s_max;
  const Row row = stopping_row(p, d, req, stop < n && !p.probs);
  int64_t v0, v1;
  run_of(p.vocab, seg * kWarps + w, v0, v1);
  double z = 0.0, held = 0.0;
  for (int64_t i0 = v0 + lane; i0 < v1; i0 += 32 * kPickBatch) {
    float l[kPickBatch];
#pragma unroll
    for (int k = 0; k < kPickBatch; ++k) l[k] = i0 + k * 32 < v1 ? __ldg(row.x + i0 + k * 32) : 0.f;
#pragma unroll
    for (int k = 0; k < kPickBatch; ++k) {
      const int64_t v = i0 + k * 32;
      if (v < v1) {
        const double e = row.weight(l[k]);
        z += e;
        if (v != row.hole) held += e;
      }
    }
  }
  z = warp_sum_d(z);
  held = warp_sum_d(held);
  if (lane == 0) {
    p.parts[(int64_t)req * kRuns + seg * kWarps + w] = make_double2(z, held);
    __threadfence();
  }
  if (d.draw == 2 && p.probs) return;
  if (last_segment(p.counters + 2 * req)) draw_index(p, req, d);
}

// Where drafts have probabilities: part[1] of a segment becomes the sum of max(p - q, 0).
__global__ void __launch_bounds__(kStatThreads) verify_rest_kernel(const VerifyArgs p) {
  griddep_launch();
  griddep_wait();
  constexpr int kWarps = kStatThreads / 32;
  __shared__ double s_z;
  const int req = (int)blockIdx.y, seg = (int)blockIdx.x;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const Decision d = p.decisions[req];
  if (d.draw != 2) return;
  Row row = stopping_row(p, d, req, true);
  if (w == 0) {
    double Z = 0.0;
#pragma unroll
    for (int k = 0; k < kRuns / 32; ++k) Z += p.parts[(int64_t)req * kRuns + k * 32 + lane].x;
    Z = warp_sum_d(Z);
    if (lane == 0) s_z = Z;
  }
  int64_t v0, v1;
  run_of(p.vocab, seg * kWarps + w, v0, v1);
  __syncthreads();
  row.inv_z = 1.0 / s_z;
  double r = 0.0;
  for (int64_t i0 = v0 + lane; i0 < v1; i0 += 32 * kPickBatch) {
    float l[kPickBatch], q[kPickBatch];
#pragma unroll
    for (int k = 0; k < kPickBatch; ++k) {
      const int64_t v = i0 + k * 32;
      l[k] = v < v1 ? __ldg(row.x + v) : 0.f;
      q[k] = v < v1 ? __ldg(row.q + v) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kPickBatch; ++k)
      if (i0 + k * 32 < v1) r += fmax(row.weight(l[k]) * row.inv_z - (double)q[k], 0.0);
  }
  r = warp_sum_d(r);
  if (lane == 0) {
    p.rest[(int64_t)req * kRuns + seg * kWarps + w] = r;
    __threadfence();
  }
  if (last_segment(p.counters + 2 * req + 1)) draw_index(p, req, d);
}

}  // namespace

extern "C" int mg_verify_workspace_bytes(int64_t rows, int64_t vocab, int b, size_t* bytes) {
  if (!bytes || rows < 0 || vocab <= 0 || b < 0) return MG_ERR_INVALID_ARG;
  if (vocab > 0x7fffffc0 || rows > 65535 || b > 65535) return MG_ERR_UNSUPPORTED;
  *bytes = (size_t)rows * (size_t)((vocab + kStatChunk - 1) / kStatChunk) * sizeof(float4) +
           (size_t)b * (sizeof(Decision) + kRuns * (sizeof(double2) + sizeof(double)) + 2 * sizeof(int32_t));
  return MG_OK;
}

extern "C" int mg_verify_drafts(const float* logits, int64_t ld, int64_t rows, int64_t vocab, const int32_t* tokens,
                                const int32_t* cu_rows, int b, const float* draft_probs, int64_t ld_probs,
                                const float* uniforms, const float* temperatures, int32_t* accepted, int32_t* next,
                                void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  const int rc = mg_verify_workspace_bytes(rows, vocab, b, &need);
  if (rc) return rc;
  if (b < 0 || ld < vocab || (draft_probs && ld_probs < vocab) ||
      (b > 0 && (!cu_rows || !accepted || !next)) || (rows > 0 && (!logits || !tokens || !uniforms)) ||
      workspace_bytes < need || (need && !workspace) || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return MG_ERR_INVALID_ARG;
  if (b == 0) return MG_OK;
  // (a request is answered while others are still at work on the inputs and on the workspace)
  const struct { const void* at; int64_t bytes; } held[] = {
      {logits, rows > 0 ? ((rows - 1) * ld + vocab) * 4 : 0}, {tokens, rows * 4}, {cu_rows, ((int64_t)b + 1) * 4},
      {draft_probs, draft_probs && rows > 0 ? ((rows - 1) * ld_probs + vocab) * 4 : 0}, {uniforms, rows * 4},
      {temperatures, temperatures ? (int64_t)b * 4 : 0}, {workspace, (int64_t)need}};
  const int64_t out_bytes = (int64_t)b * 4;
  if (mg_overlap(accepted, out_bytes, next, out_bytes)) return MG_ERR_INVALID_ARG;
  for (const auto& h : held) {
    if (h.bytes > 0 && (mg_overlap(accepted, out_bytes, h.at, h.bytes) || mg_overlap(next, out_bytes, h.at, h.bytes)))
      return MG_ERR_INVALID_ARG;
  }
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
  a.parts = reinterpret_cast<double2*>(a.stats + rows * a.chunks);
  a.decisions = reinterpret_cast<Decision*>(a.parts + (int64_t)b * kRuns);
  a.rest = reinterpret_cast<double*>(a.decisions + b);
  a.counters = reinterpret_cast<int32_t*>(a.rest + (int64_t)b * kRuns);
  a.accepted = accepted;
  a.next = next;
  cudaStream_t st = mg_stream(stream);
  if (rows > 0)
    MG_CUDA_TRY(mg_launch(verify_stats_kernel, dim3((unsigned)a.chunks, (unsigned)rows), dim3(kStatThreads), 0, st, 1, a));
  const dim3 segs(kSegments, (unsigned)b);
  MG_CUDA_TRY(mg_launch(verify_decide_kernel, segs, dim3(kStatThreads), 0, st, 1, a));
  if (draft_probs) MG_CUDA_TRY(mg_launch(verify_rest_kernel, segs, dim3(kStatThreads), 0, st, 1, a));
  MG_LAUNCH_CHECK();
  return MG_OK;
}
