// Causal attention of a ragged batch's new tokens over the paged K/V cache, from a plan (ragged_plan.cu).
//
// For request i with c cached and n new tokens, new token t (position c + t) and query head h of K/V head h / g:
//   out[t, h] = sum_{k <= c + t} softmax_k(q[t, h] . K[k] * scale) V[k]
// with K/V read through the request's block table from pools [num_blocks, hkv, 16, d], bf16 or int8 codes with one
// fp32 scale per (block, head, token) vector. n = 1 is a decoding step, n = k + 1 the verification of k drafts, and
// c = 0 a whole prompt; one launch serves any mixture of them.
//
// A work item is two tiles of 128 rows, a row being one (token, query head) of one K/V head: 128 / g tokens times g
// heads, so that the heads of a group share every K/V tile. The roles of a CTA (one per SM):
//   * a producer warp brings K and V tiles of 128 tokens (eight blocks) into a ring of shared-memory stages by TMA;
//     for an int8 cache a warpgroup reads the codes instead and stores them as bf16 (exact), already swizzled;
//   * one thread issues the tensor-core products: S = Q K^T into tensor memory, and O += P V with P read from tensor
//     memory (written over S) and V from the stage it was loaded to, taken as an MN-major operand, so that nothing is
//     transposed. The two row tiles alternate: while one's softmax runs, the other's products do;
//   * two warpgroups of softmax, one thread per row: no exchange between threads is needed for a row's maximum and
//     sum. P is rounded to bf16, the type of V (one product has one operand type); the running maximum, the sum (of
//     the unrounded values) and O are fp32. O is rescaled only when a row's maximum grew by more than 2^8 in the
//     exponentials' scale: until then exponentials up to 2^8 stay far inside the range of fp32 and bf16, and the
//     final division by the sum removes the common factor.
// An item that the plan split along the keys leaves (O, maximum, sum) in a workspace slot, and a second kernel
// merges the slots of each split item in order.
//
// Masked places: scores of keys behind a row's position are replaced before they are used, whatever they are.
// P is zero there, and 0 * V must be zero too: rows of V behind the item's last key are zeroed in the stage, and a
// V row that some of a tile's rows may not see is looked over; where one holds an infinity or a NaN, that tile's
// product is done by the softmax threads, over the keys each row sees.
#include "ragged.cuh"

namespace {

constexpr int kRows = kRagTile;

template <int D, bool Q8>
struct RagCfg {
  static constexpr int kSlab = D >= 64 ? 128 : 64;                 // bytes of a swizzled shared-memory row
  static constexpr int kSlabs = D * 2 / kSlab;                     // slabs side by side in a tile
  static constexpr int kSlabBytes = kRows * kSlab;
  static constexpr int kTileBytes = kRows * D * 2;
  static constexpr int kStages = D == 128 ? (Q8 ? 4 : 5) : (D == 64 ? 8 : 12);
  // the scales of a tile are read until its softmax is done, which the stage of K (free once S is) does not wait for:
  // a tile's K may be stored while the kStages / 2 tiles before it are still at work
  static constexpr int kScaleRing = kStages / 2 + 1;
  static constexpr int kQ = 0;
  static constexpr int kRing = 2 * kTileBytes;
  static constexpr int kScales = kRing + kStages * kTileBytes;     // [ring][K 128 | V 128] fp32
  static constexpr int kBars = kScales + (Q8 ? kScaleRing * 2 * kRows * 4 : 0);
  static constexpr int kSmem = kBars + 512 + 1024;
  static constexpr int kThreads = Q8 ? 13 * 32 : 10 * 32;
  static constexpr uint32_t kO = 256;                              // tensor-memory columns: S0, S1, O0, O1
  // fp32 accumulator, bf16 operands, M = 128; S: K-major B of N = 128; O: MN-major B of N = D
  static constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((kRows >> 3) << 17) | ((kRows >> 4) << 24);
  static constexpr uint32_t kIdescO =
      (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((kRows >> 4) << 24);
};

// Byte offset of the 16-byte chunk `c` (8 bf16) of row r in a swizzled tile.
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  if constexpr (D >= 64)
    return (uint32_t)((c >> 3) * (kRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
  else
    return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// Shared-memory operand descriptor: swizzle 128 B (rows of 128 B) or 64 B (rows of 64 B); groups of eight rows are
// 8 * row apart. lead: distance of the next swizzle-wide slab of an MN-major operand (unused for K-major).
template <int D>
__device__ __forceinline__ uint64_t rag_desc(uint32_t saddr, uint32_t lead) {
  constexpr uint32_t kGroup = D >= 64 ? 1024 : 512;
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lead >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(kGroup >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)(D >= 64 ? 2u : 4u) << 61;
  return d;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
struct RagArgs {
  const __nv_bfloat16* q;
  int64_t rows, num_blocks;
  const int32_t* tables;
  int max_blocks, b, hq, hkv, group, tok_tile, max_slots;
  float scale_log2;
  const uint8_t* work;
  int64_t list_off, merge_off;
  const int8_t *k8, *v8;
  const float *ks, *vs;
  __nv_bfloat16* out;
  float* ws_o;   // [slots][hkv][2 * 128][D]
  float2* ws_ml; // [slots][hkv][2 * 128]: maximum in log2 units, sum
};

template <int D, bool Q8>
__global__ void __launch_bounds__(RagCfg<D, Q8>::kThreads, 1)
    ragged_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                       const RagArgs p) {
  using C = RagCfg<D, Q8>;
  constexpr int NS = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* empty = full + NS;
  uint64_t* sfull = empty + NS;    // [2] a row tile's scores are in tensor memory (and its earlier P V is done)
  uint64_t* pready = sfull + 2;    // [2] its probabilities are
  uint64_t* ofull = pready + 2;    // [2] its output is complete
  uint64_t* qfull = ofull + 2;
  uint64_t* drained = qfull + 1;
  uint64_t* looked = drained + 1;  // [2] every warp of a warpgroup has looked over a masked tile's V rows
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(looked + 2);
  int* skip = reinterpret_cast<int*>(tmem_holder + 1);  // [2] the softmax threads did this tile's P V themselves
  int* odd_v = skip + 2;           // [2] an infinity or NaN was found among V rows that some row may not see

  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  const RagHead* head = reinterpret_cast<const RagHead*>(p.work);
  const int entry = (int)blockIdx.x / p.hkv, kvh = (int)blockIdx.x % p.hkv;
  if (entry >= head->n_list) return;
  const RagItem it = reinterpret_cast<const RagItem*>(p.work + p.list_off)[entry];
  if (it.row0 < 0 || (int64_t)it.row0 + it.n_tok > p.rows || it.seq < 0 || it.seq >= p.b ||
      (int64_t)it.kv_len > (int64_t)p.max_blocks * 16 || it.slot >= p.max_slots) {  // a plan for other sizes
    if (threadIdx.x == 0) mg_record_error(MG_ERR_DEVICE, 510);
    return;
  }
  // K/V tiles of each row tile: up to its last token's position (none for an empty second tile)
  int n_w[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int toks = min(p.tok_tile, it.n_tok - w * p.tok_tile);
    const int last = it.pos0 + w * p.tok_tile + toks - 1;
    n_w[w] = toks <= 0 ? 0 : max(0, min(it.kt1, last / kRows + 1) - it.kt0);
  }
  const int n_all = max(n_w[0], n_w[1]);

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], Q8 ? 128 : 1);
      mbar_init(&empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sfull[w], 1);
      mbar_init(&pready[w], 4);
      mbar_init(&ofull[w], 1);
      mbar_init(&looked[w], 4);
      skip[w] = odd_v[w] = 0;
    }
    mbar_init(qfull, 8);
    mbar_init(drained, 1);
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int32_t* table = p.tables + (int64_t)it.seq * p.max_blocks;
  const int blocks = (it.kv_len + 15) >> 4;

  if (warp >= 8) {
    if (warp == 9 && !Q8) {
      // ---------------- TMA producer: K_0, V_0, K_1, V_1, ... ----------------
      // lane = (block of the tile, slab of the row); K and V tiles of the same index use the same block ids
      const int blk = lane & 7, slab = lane >> 3;
      const bool mine = slab < C::kSlabs;
      bool ok = true;
      int i = 0;
      for (int j = 0; j < n_all && ok; ++j) {
        const int b0 = (it.kt0 + j) * 8, nb = min(8, blocks - b0);
        int row = (int)(p.num_blocks * p.hkv * 16);  // behind the pool: reads zeros
        if (blk < nb) {
          const int32_t id = table[b0 + blk];
          if (id >= 0 && id < p.num_blocks) row = (id * p.hkv + kvh) * 16;
          else mg_record_error(MG_ERR_DEVICE, 511);
        }
        for (int kv = 0; kv < 2 && ok; ++kv, ++i) {
          const int s = i % NS;
          if (i >= NS) ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((i / NS) - 1) & 1, 512));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)(nb * 16 * D * 2));
          __syncwarp();
          if (mine && blk < nb)
            tma_load_2d(smem + C::kRing + s * C::kTileBytes + slab * C::kSlabBytes + blk * 16 * C::kSlab,
                        kv ? &tv : &tk, &full[s], slab * (C::kSlab / 2), row);
        }
      }
      // the loads that were started have landed before this CTA's memory goes to another
      for (int k = max(0, i - NS); k < i; ++k) mbar_wait(&full[k % NS], (k / NS) & 1, 513);
    } else if (warp == 8) {
      // ---------------- tensor-core issue ----------------
      if (lane == 0) {
        bool ok = mbar_wait(qfull, 0, 514);
        const uint32_t sq = smem_u32(smem + C::kQ), sr = smem_u32(smem + C::kRing);
        auto scores = [&](int w, int j) {  // S_w = Q_w K_j^T
          const uint32_t a = sq + (uint32_t)(w * C::kTileBytes), k = sr + (uint32_t)((2 * j % NS) * C::kTileBytes);
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            const uint32_t off = (uint32_t)((x * 32 / C::kSlab) * C::kSlabBytes + (x * 32) % C::kSlab);
            tc_mma_ss(tmem + (uint32_t)(w * kRows), rag_desc<D>(a + off, 16), rag_desc<D>(k + off, 16), C::kIdescS,
                      x > 0);
          }
          tc_commit(&sfull[w]);
        };
        if (ok && n_all > 0) {
          ok = mbar_wait(&full[0], 0, 515);
          tc_fence_after();
          if (ok) {
            if (n_w[0] > 0) scores(0, 0);
            if (n_w[1] > 0) scores(1, 0);
            tc_commit(&empty[0]);
          }
        }
        for (int j = 0; j < n_all && ok; ++j) {
          const int sv = (2 * j + 1) % NS, sk = (2 * j + 2) % NS;
          for (int w = 0; w < 2 && ok; ++w) {
            if (j >= n_w[w]) continue;
            ok = mbar_wait(&full[sv], ((2 * j + 1) / NS) & 1, 516) && mbar_wait(&pready[w], j & 1, 517);
            if (!ok) break;
            tc_fence_after();
            if (!*(volatile int*)&skip[w]) {
              const uint32_t v = sr + (uint32_t)(sv * C::kTileBytes);
#pragma unroll
              for (int x = 0; x < kRows / 16; ++x)  // 16 keys a step: 16 rows of V
                tc_mma_ts(tmem + C::kO + (uint32_t)(w * D), tmem + (uint32_t)(w * kRows + x * 8),
                          rag_desc<D>(v + (uint32_t)(x * 16 * C::kSlab), C::kSlabBytes), C::kIdescO, j > 0 || x > 0);
            }
            if (j + 1 < n_w[w]) {
              ok = mbar_wait(&full[sk], ((2 * j + 2) / NS) & 1, 518);
              if (!ok) break;
              tc_fence_after();
              scores(w, j + 1);
            } else {
              tc_commit(&ofull[w]);
            }
          }
          if (!ok) break;
          tc_commit(&empty[sv]);
          if (j + 1 < n_all) tc_commit(&empty[sk]);
        }
        tc_commit(drained);
        mbar_wait(drained, 0, 519);
      }
    } else if (Q8 && warp >= 9) {
      // ---------------- int8 codes -> bf16 tiles ----------------
      const int t = threadIdx.x - 9 * 32;
      float* scales = reinterpret_cast<float*>(smem + C::kScales);
      constexpr int kParts = D / 16;              // 16-byte pieces of a vector of codes
      constexpr int kPer = kRows * kParts / 128;  // pieces per thread and tile
      bool ok = true;
      int i = 0;
      for (int j = 0; j < n_all && ok; ++j) {
        const int key0 = (it.kt0 + j) * kRows;
        for (int kv = 0; kv < 2 && ok; ++kv, ++i) {
          const int s = i % NS;
          const int8_t* pool = kv ? p.v8 : p.k8;
          uint4 c[kPer];
#pragma unroll
          for (int x = 0; x < kPer; ++x) {  // all loads first
            const int piece = x * 128 + t, key = key0 + piece / kParts;
            c[x] = make_uint4(0, 0, 0, 0);
            if (key < it.kv_len) {
              const int32_t id = table[key >> 4];
              if (id >= 0 && id < p.num_blocks)
                c[x] = *reinterpret_cast<const uint4*>(
                    pool + (((int64_t)id * p.hkv + kvh) * 16 + (key & 15)) * D + (piece % kParts) * 16);
              else mg_record_error(MG_ERR_DEVICE, 511);
            }
          }
          float sc = 0.f;
          if (key0 + t < it.kv_len) {
            const int32_t id = table[(key0 + t) >> 4];
            if (id >= 0 && id < p.num_blocks)
              sc = (kv ? p.vs : p.ks)[((int64_t)id * p.hkv + kvh) * 16 + ((key0 + t) & 15)];
          }
          if (i >= NS) ok = mbar_wait(&empty[s], ((i / NS) - 1) & 1, 512);
          if (!ok) break;
          uint8_t* dst = smem + C::kRing + s * C::kTileBytes;
#pragma unroll
          for (int x = 0; x < kPer; ++x) {
            const int piece = x * 128 + t, r = piece / kParts, q = (piece % kParts) * 2;
            uint4 lo, hi;
            i8x4_to_bf16x4(c[x].x, lo.x, lo.y);
            i8x4_to_bf16x4(c[x].y, lo.z, lo.w);
            i8x4_to_bf16x4(c[x].z, hi.x, hi.y);
            i8x4_to_bf16x4(c[x].w, hi.z, hi.w);
            *reinterpret_cast<uint4*>(dst + chunk_at<D>(r, q)) = lo;
            *reinterpret_cast<uint4*>(dst + chunk_at<D>(r, q + 1)) = hi;
          }
          scales[(j % C::kScaleRing) * 2 * kRows + kv * kRows + t] = sc;
          fence_async_smem();
          mbar_arrive(&full[s]);
        }
      }
    }
  } else {
    // ---------------- softmax: one thread per row ----------------
    const int w = warp >> 2, t = threadIdx.x & 127;  // row tile, row
    const int valid = max(0, min(p.tok_tile, it.n_tok - w * p.tok_tile)) * p.group;
    const int tok0 = w * p.tok_tile;
    const int64_t row_stride = (int64_t)p.hq * D;
    const int64_t base = (int64_t)(it.row0 + tok0) * row_stride + (int64_t)kvh * p.group * D;
    {  // this tile's rows of Q into shared memory (rows that are not there as zeros)
      constexpr int kChunks = D / 8;
#pragma unroll 8
      for (int x = 0; x < kRows * kChunks / 128; ++x) {
        const int idx = x * 128 + t, r = idx / kChunks, c = idx % kChunks;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < valid)
          v = *reinterpret_cast<const uint4*>(p.q + base + (int64_t)(r / p.group) * row_stride + (r % p.group) * D + c * 8);
        *reinterpret_cast<uint4*>(smem + C::kQ + w * C::kTileBytes + chunk_at<D>(r, c)) = v;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(qfull);
    }
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lane_base + (uint32_t)(w * kRows), to = tmem + lane_base + C::kO + (uint32_t)(w * D);
    const int first_pos = it.pos0 + tok0, my_pos = first_pos + t / p.group;
    const bool warp_on = (warp & 3) * 32 < valid;
    float m = -INFINITY, l = 0.f;  // m: the maximum in use, in score units
    bool ok = true;
    int looks = 0;
    for (int j = 0; j < n_w[w] && ok; ++j) {
      const int key0 = (it.kt0 + j) * kRows;
      ok = __all_sync(0xffffffffu, mbar_wait(&sfull[w], j & 1, 520));
      if (!ok) break;
      tc_fence_after();
      const bool masked = key0 + kRows - 1 > first_pos;  // some row of the tile does not see all its keys
      bool by_hand = false;
      if constexpr (!Q8) {
        if (masked) {
          // V rows that some row may not see: zero those behind the item's keys, look the others over
          const int sv = (2 * j + 1) % NS;
          ok = __all_sync(0xffffffffu, mbar_wait(&full[sv], ((2 * j + 1) / NS) & 1, 521));
          if (!ok) break;
          uint8_t* v = smem + C::kRing + sv * C::kTileBytes;
          const int r_first = max(0, first_pos + 1 - key0), r_end = min(kRows, it.kv_len - key0);
          bool odd = false;
          for (int x = r_first * (D / 8) + t; x < kRows * (D / 8); x += 128) {
            const int r = x / (D / 8);
            uint4* at = reinterpret_cast<uint4*>(v + chunk_at<D>(r, x % (D / 8)));
            if (r >= r_end) {
              *at = make_uint4(0, 0, 0, 0);
            } else {
              const uint4 q = *at;
              const uint32_t e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
              for (int y = 0; y < 4; ++y)
                odd |= (e[y] & 0x7f800000u) == 0x7f800000u || (e[y] & 0x7f80u) == 0x7f80u;
            }
          }
          fence_async_smem();
          // (any thread's finding is every thread's; once found it holds for the item's later tiles too)
          odd = __any_sync(0xffffffffu, odd);
          if (lane == 0) {
            if (odd) *(volatile int*)&odd_v[w] = 1;
            mbar_arrive(&looked[w]);
          }
          ok = __all_sync(0xffffffffu, mbar_wait(&looked[w], looks & 1, 523));
          ++looks;
          if (!ok) break;
          by_hand = *(volatile int*)&odd_v[w] != 0;
        }
      }
      if (warp_on) {
        float s[kRows];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
        tc_wait_ld();
        const float* sc = reinterpret_cast<const float*>(smem + C::kScales) + (j % C::kScaleRing) * 2 * kRows;
        if constexpr (Q8) {
#pragma unroll
          for (int c = 0; c < kRows; c += 4) {
            const float4 f = *reinterpret_cast<const float4*>(sc + c);
            s[c] *= f.x, s[c + 1] *= f.y, s[c + 2] *= f.z, s[c + 3] *= f.w;
          }
        }
        const int see = my_pos - key0;  // keys 0 .. see of the tile are this row's
        if (masked) {
#pragma unroll
          for (int c = 0; c < kRows; ++c) s[c] = c <= see ? s[c] : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int c = 1; c < kRows; ++c) mx = fmaxf(mx, s[c]);
        float m_new = fmaxf(m, mx);
        const bool grow = m == -INFINITY || (m_new - m) * p.scale_log2 > 8.f;
        if (!grow) m_new = m;
        if (__any_sync(0xffffffffu, grow) && j > 0) {
          const float f = m == -INFINITY ? 0.f : ex2((m - m_new) * p.scale_log2);
          l *= f;
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(to + c, o);
            tc_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
            tmem_st32(to + c, o);
          }
          tc_wait_st();
        }
        m = m_new;
        const float off = m == -INFINITY ? 0.f : m * p.scale_log2;
        float sum = 0.f;
        uint32_t pk[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            float a = ex2(fmaf(s[h * 64 + c], p.scale_log2, -off)), b = ex2(fmaf(s[h * 64 + c + 1], p.scale_log2, -off));
            sum += a + b;
            if constexpr (Q8) {  // the value's scale, with nothing of a masked key's
              a = !masked || h * 64 + c <= see ? a * sc[kRows + h * 64 + c] : 0.f;
              b = !masked || h * 64 + c + 1 <= see ? b * sc[kRows + h * 64 + c + 1] : 0.f;
            }
            pk[c / 2] = pack_bf16x2(a, b);
          }
          tmem_st32(ts + h * 32, pk);
        }
        l += sum;
        tc_wait_st();
        if constexpr (!Q8) {
          if (by_hand) {
            // O += P V over the keys that each row sees, from the stage, in the tensor cores' place
            const uint8_t* v = smem + C::kRing + ((2 * j + 1) % NS) * C::kTileBytes;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              if (j > 0) {
                tmem_ld32(to + c, o);
                tc_wait_ld();
              } else {
#pragma unroll
                for (int x = 0; x < 32; ++x) o[x] = 0;
              }
#pragma unroll 1
              for (int k = 0; k < kRows; k += 64) {
                uint32_t pr[32];
                tmem_ld32(ts + k / 2, pr);
                tc_wait_ld();
#pragma unroll
                for (int kk = 0; kk < 64; ++kk) {
                  const float pv = kk & 1 ? bf16hi(pr[kk / 2]) : bf16lo(pr[kk / 2]);
                  if (k + kk <= see) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                      const uint4 q = *reinterpret_cast<const uint4*>(v + chunk_at<D>(k + kk, c / 8 + x));
                      const uint32_t e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                      for (int y = 0; y < 4; ++y) {
                        o[x * 8 + 2 * y] = __float_as_uint(fmaf(pv, bf16lo(e[y]), __uint_as_float(o[x * 8 + 2 * y])));
                        o[x * 8 + 2 * y + 1] =
                            __float_as_uint(fmaf(pv, bf16hi(e[y]), __uint_as_float(o[x * 8 + 2 * y + 1])));
                      }
                    }
                  }
                }
              }
              tmem_st32(to + c, o);
            }
            tc_wait_st();
          }
        }
      }
      if (t == 0) *(volatile int*)&skip[w] = by_hand;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pready[w]);
    }
    // ---------------- epilogue ----------------
    if (n_w[w] > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(&ofull[w], 0, 522));
    if (warp_on) {
      tc_fence_after();
      const bool any = n_w[w] > 0 && ok;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t slot_row = ((int64_t)it.slot * p.hkv + kvh) * (2 * kRows) + w * kRows + t;
      __nv_bfloat16* dst = p.out + base + (int64_t)(t / p.group) * row_stride + (t % p.group) * D;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (any) {
          tmem_ld32(to + c, o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = 0;
        }
        if (t < valid) {
          if (it.slot < 0) {
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
              uint4 v;
              v.x = pack_bf16x2(__uint_as_float(o[x]) * inv, __uint_as_float(o[x + 1]) * inv);
              v.y = pack_bf16x2(__uint_as_float(o[x + 2]) * inv, __uint_as_float(o[x + 3]) * inv);
              v.z = pack_bf16x2(__uint_as_float(o[x + 4]) * inv, __uint_as_float(o[x + 5]) * inv);
              v.w = pack_bf16x2(__uint_as_float(o[x + 6]) * inv, __uint_as_float(o[x + 7]) * inv);
              *reinterpret_cast<uint4*>(dst + c + x) = v;
            }
          } else {
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<uint4*>(p.ws_o + slot_row * D + c + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
          }
        }
      }
      if (it.slot >= 0 && t < valid)
        p.ws_ml[slot_row] = make_float2(any && m != -INFINITY ? m * p.scale_log2 : -INFINITY, any ? l : 0.f);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Merge of the partial states of the items that were split: row r of item m, in slot order,
//   M = max m_s,  out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.
// One warp per row at a time; d / 32 columns per lane.
constexpr int kMergeWarps = 8;

template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) ragged_merge_kernel(const RagArgs p) {
  griddep_launch();
  griddep_wait();
  const RagHead* head = reinterpret_cast<const RagHead*>(p.work);
  const int m = (int)blockIdx.x, kvh = (int)blockIdx.y;
  if (m >= head->n_merge) return;
  const RagMerge g = reinterpret_cast<const RagMerge*>(p.work + p.merge_off)[m];
  if (g.row0 < 0 || (int64_t)g.row0 + g.n_tok > p.rows || g.slot0 < 0 || g.slot0 + g.parts > p.max_slots) return;  // (the attention kernel has recorded it)
  const int lane = threadIdx.x & 31, rows = g.n_tok * p.group;
  for (int r = (int)(blockIdx.z * kMergeWarps + (threadIdx.x >> 5)); r < rows; r += (int)gridDim.z * kMergeWarps) {
    // row r of the item is (token r / group, head r % group); its place in the two tiles
    const int tok = r / p.group, w = tok / p.tok_tile;
    const int at = w * kRows + r - w * p.tok_tile * p.group;
    const int64_t first = ((int64_t)g.slot0 * p.hkv + kvh) * (2 * kRows) + at, step = (int64_t)p.hkv * (2 * kRows);
    float M = -INFINITY;
    for (int s = lane; s < g.parts; s += 32) M = fmaxf(M, p.ws_ml[first + s * step].x);
    M = warp_max(M);
    float L = 0.f, o[D / 32] = {};
    for (int s = 0; s < g.parts; ++s) {
      const float2 ml = p.ws_ml[first + s * step];
      const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
      L += f * ml.y;
      const float* src = p.ws_o + (first + s * step) * D + lane * (D / 32);
#pragma unroll
      for (int x = 0; x < D / 32; ++x) o[x] += f == 0.f ? 0.f : f * src[x];
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    __nv_bfloat16* dst = p.out + (int64_t)(g.row0 + tok) * p.hq * D + ((int64_t)kvh * p.group + r % p.group) * D + lane * (D / 32);
#pragma unroll
    for (int x = 0; x < D / 32; ++x) dst[x] = __float2bfloat16_rn(o[x] * inv);
  }
}

template <int D, bool Q8>
int launch_ragged(const RagArgs& a, const RagShape& s, const void* k_pool, const void* v_pool, cudaStream_t st) {
  using C = RagCfg<D, Q8>;
  static bool done[64] = {};
  static std::mutex mu;
  MG_CUDA_TRY(mg_once_per_device(done, mu, [] {
    return cudaFuncSetAttribute(ragged_attn_kernel<D, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  }));
  CUtensorMap tk{}, tv{};
  if constexpr (!Q8) {
    const uint64_t rows = (uint64_t)a.num_blocks * a.hkv * 16;
    if (rows > 0x7fffffffull) return MG_ERR_UNSUPPORTED;
    const CUtensorMapSwizzle sw = D >= 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    int rc = mg_make_map_2d(&tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, k_pool, D, rows, D * 2, C::kSlab / 2, 16, sw);
    if (rc == MG_OK) rc = mg_make_map_2d(&tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, v_pool, D, rows, D * 2, C::kSlab / 2, 16, sw);
    if (rc) return rc;
  }
  const int64_t ctas = s.max_list * a.hkv;
  if (ctas > 0x7fffffff || a.hkv > 65535) return MG_ERR_UNSUPPORTED;
  MG_CUDA_TRY(mg_launch(ragged_attn_kernel<D, Q8>, dim3((unsigned)ctas), dim3(C::kThreads), C::kSmem, st, 1, tk, tv, a));
  MG_CUDA_TRY(mg_launch(ragged_merge_kernel<D>, dim3((unsigned)s.max_merges, (unsigned)a.hkv, 8), dim3(kMergeWarps * 32),
                        0, st, 1, a));
  MG_LAUNCH_CHECK();
  return MG_OK;
}

}  // namespace

extern "C" int mg_ragged_attn_workspace_bytes(int64_t max_rows, int b, int hq, int hkv, int d, size_t* bytes) {
  if (!bytes || max_rows < 0 || b < 0 || hq <= 0 || hkv <= 0 || hq % hkv) return MG_ERR_INVALID_ARG;
  RagShape s;
  if (!rag_shape(max_rows, b, hq, hkv, d, mg_sm_count(), &s)) return MG_ERR_UNSUPPORTED;
  *bytes = (size_t)s.max_slots * hkv * 2 * kRows * (d * sizeof(float) + sizeof(float2));
  return MG_OK;
}

extern "C" int mg_ragged_attn(const void* q, int64_t rows, const void* k_pool, const void* v_pool,
                              const float* k_scales, const float* v_scales, int64_t num_blocks,
                              const int32_t* block_tables, int max_blocks, int b, int64_t max_rows, int hq, int hkv,
                              int d, float scale, const void* work, void* out, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const bool q8 = k_scales != nullptr;
  if (rows < 0 || b < 0 || max_rows < 0 || hq <= 0 || hkv <= 0 || hq % hkv || max_blocks <= 0 || num_blocks <= 0 ||
      num_blocks > (1 << 27) || !(scale > 0.f) || scale > 1e30f || q8 != (v_scales != nullptr))
    return MG_ERR_INVALID_ARG;
  RagShape s;
  if (!rag_shape(max_rows, b, hq, hkv, d, mg_sm_count(), &s)) return MG_ERR_UNSUPPORTED;
  if (rows == 0 || b == 0 || max_rows == 0) return MG_OK;
  size_t need = 0;
  const int rc = mg_ragged_attn_workspace_bytes(max_rows, b, hq, hkv, d, &need);
  if (rc) return rc;
  if (!q || !k_pool || !v_pool || !block_tables || !work || !out || !workspace || workspace_bytes < need)
    return MG_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool) |
       reinterpret_cast<uintptr_t>(work) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return MG_ERR_INVALID_ARG;
  RagArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.rows = rows;
  a.num_blocks = num_blocks;
  a.tables = block_tables;
  a.max_blocks = max_blocks;
  a.b = b;
  a.hq = hq;
  a.hkv = hkv;
  a.group = s.group;
  a.tok_tile = s.tok_tile;
  a.max_slots = s.max_slots;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.work = static_cast<const uint8_t*>(work);
  a.list_off = s.list_off;
  a.merge_off = s.merge_off;
  a.k8 = static_cast<const int8_t*>(k_pool);
  a.v8 = static_cast<const int8_t*>(v_pool);
  a.ks = k_scales;
  a.vs = v_scales;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ws_o = static_cast<float*>(workspace);
  a.ws_ml = reinterpret_cast<float2*>(a.ws_o + (size_t)s.max_slots * hkv * 2 * kRows * d);
  cudaStream_t st = mg_stream(stream);
  if (q8) {
    if (d == 32) return launch_ragged<32, true>(a, s, k_pool, v_pool, st);
    return d == 64 ? launch_ragged<64, true>(a, s, k_pool, v_pool, st) : launch_ragged<128, true>(a, s, k_pool, v_pool, st);
  }
  if (d == 32) return launch_ragged<32, false>(a, s, k_pool, v_pool, st);
  return d == 64 ? launch_ragged<64, false>(a, s, k_pool, v_pool, st) : launch_ragged<128, false>(a, s, k_pool, v_pool, st);
}
