// The plan of one step over a ragged batch: request i brings q_lens[i] new tokens on top of ctx_lens[i] cached
// ones. With kv = ctx + q, need = ceil(kv / 16) blocks and cu = the exclusive prefix sum of q:
//   * the blocks a table lacks, need - held, come off the free list in request order;
//   * row r of request i (cu[i] <= r < cu[i+1]) stands at position p = ctx[i] + r - cu[i] and its K/V go to slot
//     table[i][p / 16] * 16 + p % 16;
//   * the attention's work list: every request's rows in items of two row tiles, longest first, an item whose
//     keys are more than one SM's share of the whole split along the keys.
//
// A few kilobytes of integers: what bounds it is the launch and the chain of dependent memory round trips
// (lengths -> prefix sums -> table entries -> stores), not bandwidth. So every CTA of one cluster reads all the
// lengths and scans them for itself instead of waiting for another CTA's scan, rank 0 builds the work list while
// the others write the rows, and one cluster barrier separates reading the inputs from writing the outputs,
// which may therefore alias them (a loop feeds held-block counts, the cursor and lengths back in).
// On a B200: 9 us a call for 32 requests (6 in a graph), 15 (12) for 1000 prompts of 53 thousand rows.
#include "ragged.cuh"

int mg_sm_count() {
  static int count[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!count[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    count[dev] = n;
  }
  return count[dev];
}

namespace {

constexpr int kPlanCtas = 8;       // one cluster
constexpr int kPlanMaxB = 8192;
constexpr int kBuckets = 1024;     // work-list lengths are ordered to this resolution

struct PlanArgs {
  const int32_t *q_lens, *ctx_lens, *held, *free_blocks, *cursor;
  int32_t* tables;
  int32_t *cu, *kv_lens, *positions, *slots, *seq_ids, *held_out, *cursor_out;
  uint8_t* work;
  int64_t n_free, num_blocks, max_rows;
  int b, max_blocks, hq, hkv;
  RagShape s;
};

__device__ __forceinline__ void write_head(const PlanArgs& p, int64_t n_list, int64_t n_merge, int64_t rows) {
  RagHead h;
  h.n_list = (int32_t)n_list;
  h.n_merge = (int32_t)n_merge;
  h.rows = (int32_t)rows;
  h.max_blocks = p.max_blocks;
  h.max_rows = (int32_t)p.max_rows;
  h.b = p.b;
  h.hq = p.hq;
  h.hkv = p.hkv;
  *reinterpret_cast<RagHead*>(p.work) = h;
}

// Exclusive prefixes of N values per thread over the CTA's kT threads, in one round of barriers; total gets the sums.
// red: N * 33 words of shared memory, free for reuse after the next barrier.
template <int kT, int N>
__device__ __forceinline__ void block_prefix(int64_t (&v)[N], int64_t (*red)[33], int64_t (&total)[N]) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int64_t x[N];
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = v[n];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x[n], o);
      if (lane >= o) x[n] += y;
    }
  }
  __syncthreads();
  if (lane == 31) {
#pragma unroll
    for (int n = 0; n < N; ++n) red[n][w] = x[n];
  }
  __syncthreads();
  // every warp scans the warps' sums for itself
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int64_t s = lane < kT / 32 ? red[n][lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t z = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += z;
    }
    total[n] = __shfl_sync(0xffffffffu, s, 31);
    const int64_t before = __shfl_sync(0xffffffffu, s, w > 0 ? w - 1 : 0);
    v[n] = (w > 0 ? before : 0) + x[n] - v[n];
  }
}

// Item (i, j): tokens [j * tok_item, ...) of request i. Index of the request that owns flat item k (first[] is
// the exclusive prefix of the requests' item counts) or, with cu[], of row k.
__device__ __forceinline__ int owner(const int32_t* first, int b, int k) {
  int lo = 0, hi = b;  // first[lo] <= k < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= k) lo = mid; else hi = mid;
  }
  return lo;
}

template <int kT>
__global__ void __launch_bounds__(kT) plan_kernel(const PlanArgs p) {
  extern __shared__ int32_t sm[];
  __shared__ int64_t red[3][33];
  __shared__ int32_t hist[kBuckets];
  __shared__ int s_bad;
  int32_t* cu = sm;                    // [b + 1]
  int32_t* ctx = cu + p.b + 1;         // [b]
  int32_t* held = ctx + p.b;           // [b] blocks in the table before this step
  int32_t* take = held + p.b;          // [b] blocks taken off the free list by the requests before
  int32_t* first = take + p.b;         // [b + 1] items of the requests before
  griddep_launch();
  griddep_wait();
  const int t = threadIdx.x, rank = (int)blockIdx.x;
  if (t == 0) s_bad = 0;
  __syncthreads();

  // ---- read and scan (every CTA for itself) ----
  const int per = (p.b + kT - 1) / kT;
  const int cursor = p.cursor ? *p.cursor : 0;
  int64_t rows = 0, fresh = 0, items = 0;
  int bad = cursor < 0 ? 501 : 0;
  for (int k = 0; k < per; ++k) {
    const int i = t * per + k;
    if (i >= p.b) break;
    const int q = p.q_lens[i], c = p.ctx_lens[i];
    int h = 0, f = 0;
    if (q < 0 || c < 0 || q > p.max_rows || (int64_t)c + q > (int64_t)p.max_blocks * 16) {
      bad = 500;
    } else {
      const int need = (c + q + 15) >> 4;
      h = need;
      if (p.free_blocks) {
        h = p.held ? p.held[i] : (c + 15) >> 4;
        if (h < (c + 15) >> 4 || h > p.max_blocks) bad = 502;
        f = need > h ? need - h : 0;
      } else if (p.held) {
        h = p.held[i];
        if (h < need || h > p.max_blocks) bad = 502;
      }
      rows += q;
      fresh += f;
      items += (q + p.s.tok_item - 1) / p.s.tok_item;
    }
    ctx[i] = c;
    held[i] = h;
  }
  int64_t first3[3] = {rows, fresh, items}, all3[3];
  block_prefix<kT>(first3, red, all3);
  const int64_t n_rows = all3[0], n_fresh = all3[1], n_items = all3[2];
  int64_t r0 = first3[0], f0 = first3[1], i0 = first3[2];
  if (n_rows > p.max_rows) bad = 503;
  if (p.free_blocks && n_fresh > p.n_free - cursor) bad = 504;
  if (bad) atomicMax(&s_bad, bad);
  for (int k = 0; k < per; ++k) {
    const int i = t * per + k;
    if (i >= p.b) break;
    cu[i] = (int32_t)r0;
    take[i] = (int32_t)f0;
    first[i] = (int32_t)i0;
    const int q = p.q_lens[i], need = (ctx[i] + q + 15) >> 4;
    r0 += q;
    f0 += need > held[i] ? need - held[i] : 0;
    i0 += (q + p.s.tok_item - 1) / p.s.tok_item;
  }
  if (t == 0) {
    cu[p.b] = (int32_t)n_rows;
    first[p.b] = (int32_t)n_items;
  }
  cluster_sync_all();  // (also a barrier of this CTA) every CTA has read every input
  if (s_bad) {
    // an impossible request: an empty plan, tables and free list as they were, and the error word set
    if (t == 0 && rank == 0) mg_record_error(MG_ERR_DEVICE, s_bad);
    const int64_t g = (int64_t)rank * kT + t, step = (int64_t)kPlanCtas * kT;
    for (int64_t i = g; i <= p.b; i += step) {
      p.cu[i] = 0;
      if (i < p.b) {
        p.kv_lens[i] = 0;
        if (p.held && p.held_out != p.held) p.held_out[i] = p.held[i];
        // (not held[i]: that is what the step would have needed where there is no free list)
        if (!p.held) p.held_out[i] = ctx[i] > 0 ? (int32_t)(((int64_t)ctx[i] + 15) >> 4) : 0;
      }
    }
    for (int64_t r = g; r < p.max_rows; r += step) {
      p.positions[r] = 0;
      p.slots[r] = -1;
      p.seq_ids[r] = -1;
    }
    if (g == 0) {
      *p.cursor_out = cursor;
      write_head(p, 0, 0, 0);
    }
    return;
  }

  // ---- rank 0: per-request outputs and the work list; the other ranks: rows and new table entries ----
  if (rank == 0) {
    for (int i = t; i <= p.b; i += kT) {
      p.cu[i] = cu[i];
      if (i < p.b) {
        const int kv = ctx[i] + cu[i + 1] - cu[i], need = (kv + 15) >> 4;
        p.kv_lens[i] = kv;
        p.held_out[i] = need > held[i] ? need : held[i];
      }
    }
    if (t == 0) *p.cursor_out = cursor + (int32_t)n_fresh;

    // K/V tiles of item k and, at `share` tiles per entry, its entries
    const int n = (int)n_items;
    auto tiles = [&](int k, int& seq, int& tok0, int& cnt) {
      seq = owner(first, p.b, k);
      const int q = cu[seq + 1] - cu[seq];
      tok0 = (k - first[seq]) * p.s.tok_item;
      cnt = min(p.s.tok_item, q - tok0);
      return (ctx[seq] + tok0 + cnt + kRagTile - 1) / kRagTile;
    };
    const int ipt = (n + kT - 1) / kT;
    int64_t one[1] = {0}, total[1];
    for (int k = t * ipt; k < min(n, (t + 1) * ipt); ++k) {
      int a, c, e;
      one[0] += tiles(k, a, c, e);
    }
    block_prefix<kT>(one, red, total);
    // one SM's share; where fewer items than SMs would give entries for barely more than one wave, longer shares until
    // they fit it
    const int64_t slots_all = p.s.max_merges;
    int64_t share = (total[0] + slots_all - 1) / slots_all;
    if (share < 2) share = 2;
    for (int tries = 0; n < slots_all && tries < 24; ++tries) {
      one[0] = 0;
      for (int k = t * ipt; k < min(n, (t + 1) * ipt); ++k) {
        int a, c, e;
        one[0] += (tiles(k, a, c, e) + share - 1) / share;
      }
      block_prefix<kT>(one, red, total);
      if (total[0] <= slots_all) break;
      share += share / 8 + 1;
    }
    // merges and partial slots before this thread's items
    int64_t two[2] = {0, 0}, both[2];
    for (int k = t; k < kBuckets; k += kT) hist[k] = 0;
    for (int k = t * ipt; k < min(n, (t + 1) * ipt); ++k) {
      int a, c, e;
      const int64_t parts = (tiles(k, a, c, e) + share - 1) / share;
      if (parts > 1) {
        ++two[0];
        two[1] += parts;
      }
    }
    block_prefix<kT>(two, red, both);  // (its barriers also separate clearing the buckets from counting into them)
    int64_t merge0 = two[0], slot0 = two[1];
    const int64_t n_merge = both[0];
    // counting sort, longest entries first (the order decides only when an entry runs)
    auto bucket = [&](int64_t len) { return kBuckets - 1 - (int)(len * (kBuckets - 1) / share); };
    for (int k = t * ipt; k < min(n, (t + 1) * ipt); ++k) {
      int a, c, e;
      const int64_t nt = tiles(k, a, c, e), parts = (nt + share - 1) / share, step = (nt + parts - 1) / parts;
      for (int64_t x = 0; x < nt; x += step) atomicAdd(&hist[bucket(min(step, nt - x))], 1);
    }
    __syncthreads();
    constexpr int kPer = kBuckets / kT;  // adjacent buckets of a thread
    one[0] = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) one[0] += hist[t * kPer + k];
    block_prefix<kT>(one, red, total);
    const int64_t entries = total[0];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int c = hist[t * kPer + k];
      hist[t * kPer + k] = (int32_t)one[0];
      one[0] += c;
    }
    __syncthreads();
    RagItem* list = reinterpret_cast<RagItem*>(p.work + p.s.list_off);
    RagMerge* merges = reinterpret_cast<RagMerge*>(p.work + p.s.merge_off);
    for (int k = t * ipt; k < min(n, (t + 1) * ipt); ++k) {
      int seq, tok0, ntok;
      const int64_t nt = tiles(k, seq, tok0, ntok), parts = (nt + share - 1) / share, step = (nt + parts - 1) / parts;
      RagItem it;
      it.seq = seq;
      it.row0 = cu[seq] + tok0;
      it.n_tok = ntok;
      it.pos0 = ctx[seq] + tok0;
      it.kv_len = ctx[seq] + tok0 + ntok;
      if (parts > 1) {
        RagMerge m;
        m.row0 = it.row0;
        m.n_tok = ntok;
        m.slot0 = (int32_t)slot0;
        m.parts = (int32_t)((nt + step - 1) / step);
        merges[merge0++] = m;
      }
      int64_t x = 0;
      for (int j = 0; x < nt; x += step, ++j) {
        const int64_t len = min(step, nt - x);
        it.kt0 = (int32_t)x;
        it.kt1 = (int32_t)(x + len);
        it.slot = parts > 1 ? (int32_t)slot0 + j : -1;
        list[atomicAdd(&hist[bucket(len)], 1)] = it;
      }
      if (parts > 1) slot0 += parts;
    }
    if (t == 0) write_head(p, entries, n_merge, n_rows);
    return;
  }
  const int64_t g = (int64_t)(rank - 1) * kT + t, step = (int64_t)(kPlanCtas - 1) * kT;
  for (int64_t r = g; r < p.max_rows; r += step) {
    int pos = 0, slot = -1, seq = -1;
    if (r < n_rows) {
      seq = owner(cu, p.b, (int)r);
      pos = ctx[seq] + (int)r - cu[seq];
      const int lb = pos >> 4;
      const int32_t id = lb < held[seq] ? p.tables[(int64_t)seq * p.max_blocks + lb]
                                        : p.free_blocks[(int64_t)cursor + take[seq] + lb - held[seq]];
      if (id < 0 || id >= p.num_blocks) mg_record_error(MG_ERR_DEVICE, 505);
      else slot = id * 16 + (pos & 15);
    }
    p.positions[r] = pos;
    p.slots[r] = slot;
    p.seq_ids[r] = seq;
  }
  if (p.free_blocks && n_fresh > 0) {
    for (int64_t i = g >> 5; i < p.b; i += step >> 5) {
      const int need = (ctx[i] + cu[i + 1] - cu[i] + 15) >> 4;
      for (int lb = held[i] + (t & 31); lb < need; lb += 32)
        p.tables[i * p.max_blocks + lb] = p.free_blocks[(int64_t)cursor + take[i] + lb - held[i]];
    }
  }
}

}  // namespace

extern "C" int mg_ragged_plan_bytes(int64_t max_rows, int b, int hq, int hkv, int d, size_t* bytes) {
  if (!bytes || max_rows < 0 || b < 0 || hq <= 0 || hkv <= 0 || hq % hkv) return MG_ERR_INVALID_ARG;
  RagShape s;
  if (b > kPlanMaxB || !rag_shape(max_rows, b, hq, hkv, d, mg_sm_count(), &s)) return MG_ERR_UNSUPPORTED;
  *bytes = (size_t)s.total;
  return MG_OK;
}

extern "C" int mg_ragged_plan(const int32_t* q_lens, const int32_t* ctx_lens, int b, int64_t max_rows,
                              int32_t* block_tables, int max_blocks, int64_t num_blocks, const int32_t* held_blocks,
                              const int32_t* free_blocks, int64_t n_free, const int32_t* cursor, int hq, int hkv,
                              int d, int32_t* cu_rows, int32_t* kv_lens, int32_t* positions, int32_t* slots,
                              int32_t* seq_ids, int32_t* held_out, int32_t* cursor_out, void* work,
                              size_t work_bytes, void* stream) {
  if (b < 0 || max_rows < 0 || max_blocks <= 0 || num_blocks <= 0 || num_blocks > (1 << 27) || n_free < 0 ||
      hq <= 0 || hkv <= 0 || hq % hkv || !cu_rows || !cursor_out || !work ||
      (b > 0 && (!q_lens || !ctx_lens || !block_tables || !kv_lens || !held_out)) ||
      (max_rows > 0 && (!positions || !slots || !seq_ids)) || (reinterpret_cast<uintptr_t>(work) & 15))
    return MG_ERR_INVALID_ARG;
  PlanArgs a{};
  if (b > kPlanMaxB || max_blocks > (1 << 26) || n_free > 0x7fffffff) return MG_ERR_UNSUPPORTED;
  if (!rag_shape(max_rows, b, hq, hkv, d, mg_sm_count(), &a.s)) return MG_ERR_UNSUPPORTED;
  if (work_bytes < (size_t)a.s.total) return MG_ERR_INVALID_ARG;
  a.q_lens = q_lens;
  a.ctx_lens = ctx_lens;
  a.held = held_blocks;
  a.free_blocks = free_blocks;
  a.cursor = free_blocks ? cursor : nullptr;
  a.tables = block_tables;
  a.cu = cu_rows;
  a.kv_lens = kv_lens;
  a.positions = positions;
  a.slots = slots;
  a.seq_ids = seq_ids;
  a.held_out = held_out;
  a.cursor_out = cursor_out;
  a.work = static_cast<uint8_t*>(work);
  a.n_free = n_free;
  a.num_blocks = num_blocks;
  a.max_rows = max_rows;
  a.b = b;
  a.max_blocks = max_blocks;
  a.hq = hq;
  a.hkv = hkv;
  const size_t smem = ((size_t)5 * b + 2) * sizeof(int32_t);
  static bool done[64] = {};
  static std::mutex mu;
  MG_CUDA_TRY(mg_once_per_device(done, mu, [] {
    const int most = (5 * kPlanMaxB + 2) * (int)sizeof(int32_t);
    cudaError_t e = cudaFuncSetAttribute(plan_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    return e != cudaSuccess
               ? e
               : cudaFuncSetAttribute(plan_kernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  }));
  // Small steps are a chain of barriers, which fewer threads pass faster; with many requests a thread's share of them, one
  // behind another, costs more than the barriers. Measured in us, 256 threads against 1024: 32 requests 5.7 / 8.0, 256
  // requests 6.8 / 8.8 (1 or 16 rows each), 257 requests 9.5 / 9.1, 512 10.3 / 9.7, 1000 18.2 / 12.1. Rows matter less: 40
  // requests of 4096 rows in all 5.9 / 8.1, of 16000 7.3 / 8.4, 1000 of 53000 25.6 / 12.2; the line at 4096 keeps long lists
  // of rows and items on many threads, at the cost of up to 2 us where few requests bring them.
  if (b <= 256 && max_rows <= 4096)
    MG_CUDA_TRY(mg_launch(plan_kernel<256>, dim3(kPlanCtas), dim3(256), smem, mg_stream(stream), kPlanCtas, a));
  else
    MG_CUDA_TRY(mg_launch(plan_kernel<1024>, dim3(kPlanCtas), dim3(1024), smem, mg_stream(stream), kPlanCtas, a));
  MG_LAUNCH_CHECK();
  return MG_OK;
}
