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
//     sum. P is rounded to bf16, the type of V (one product has one operand type), over an int8 cache P times the
//     value's scale (the codes are exact in bf16); the running maximum, the sum (of the unrounded values) and O are fp32. O is rescaled only when a row's maximum grew by more than 2^8 in the
//     exponentials' scale: until then exponentials up to 2^8 stay far inside the range of fp32 and bf16, and the
//     final division by the sum removes the common factor.
// A CTA takes several items, dealt out by length, and its K/V and Q loads run ahead into the next one. An item of one row
// tile (single tokens, short drafts, a prompt's end) gives its K/V tiles to the two warpgroups in turn; the first merges
// their two states from tensor memory. An item that the plan split along the keys leaves (O, maximum, sum) in a workspace
// slot, and a second kernel merges the slots of each split item in order.
//
// Masked places: scores of keys behind a row's position are replaced before they are used, whatever they are. P is zero
// there, and 0 * V must be zero too: rows of V behind the item's last key are zeroed in the stage. What an infinity or a
// NaN in the V of a masked key would leave in the output shows there as one: a piece of work whose output holds any is
// done over in a second pass, which looks over the V rows that some row may not see, and in a tile with such a value
// leaves the product to the softmax threads, over the keys each row sees. A NaN that a row does see (in its query, in K or V)
// makes its output NaN, and so does a row of nothing but -inf.
//
// What bounds it, on a B200 (24/8 heads of 128 unless said; floors at 6.55 TB/s and 1675 TFLOP/s):
//   * an 8192-token prompt, 430 us (380-450 with the clock), 0.96 PFLOP/s, floor 246: a row tile takes its softmax (2.0 k
//     cycles, two warpgroups sharing an SM's exponentials) and then its own two products (1.0 k); the two row tiles
//     overlap to 3.2 k cycles, of which the products of both fill two thirds. Tried and slower: the products of each row
//     tile from a warp of its own (they interleave, and both softmaxes wait for both; a fifth), steps of 64 keys with two
//     score buffers (a third), reading the scores from tensor memory twice instead of holding 128 of them (up to a
//     tenth). A part of the exponentials as polynomials, and the rescaling of O behind them, gained nothing;
//   * 32 requests of 5 tokens over 300 to 4000 cached ones, 58 us, floor 35: the longest CTA's share is 1.2 times the mean,
//     and the merge adds 5 (60 with all loads from one warp, whose 2 KB copies do not start fast enough);
//   * one token over 32763, 37 us, floor 21: 8 tiles a CTA, so that the start, the first loads and the merge weigh as much;
//   * 24 packed prompts of 18 to 2005 tokens, 14/2 heads of 64, 65 us: the exponentials of whole 128 x 128 tiles, most of
//     them cut by the diagonal (their pipe is busy 44 % of the time); the products would take 13. (128 columns of tensor
//     memory are not used at this head size; the figures above for other ways were taken at heads of 128.)
//   * 16 chunks over up to 3800 cached tokens, bf16, 59 us: two or three short items a CTA, each with an end of its own;
//     int8, 83: codes to bf16 by one warpgroup (2.0 k cycles a tile) and a softmax of 4.2 k cycles, the scales'
//     products included, in code that strains the instruction caches (95 while all of it was unrolled, with a row per
//     thread).
#include <type_traits>

#include "ragged.cuh"

namespace {

constexpr int kRows = kRagTile;

template <int D, bool Q8>
struct RagCfg {
  static constexpr int kSlab = D >= 64 ? 128 : 64;                 // bytes of a swizzled shared-memory row
  static constexpr int kSlabs = D * 2 / kSlab;                     // slabs side by side in a tile
  static constexpr int kSlabBytes = kRows * kSlab;
  static constexpr int kTileBytes = kRows * D * 2;
  static constexpr int kStages = D == 128 ? (Q8 ? 3 : 5) : (D == 64 ? 6 : 8);
  static constexpr int kCodeStages = Q8 ? (D == 128 ? 3 : 4) : 0;  // int8 codes on their way to a stage
  static constexpr int kCodeBytes = kRows * D;
  // the scales of a tile are read until its softmax is done, which the stage of K (free once S is) does not wait for:
  // a tile's K may be stored while the kStages / 2 tiles before it are still at work
  static constexpr int kScaleRing = kStages / 2 + 1;
  static constexpr int kRing = 2 * kTileBytes;                     // (the two tiles of Q come first)
  static constexpr int kCodes = kRing + kStages * kTileBytes;
  static constexpr int kCodeScales = kCodes + kCodeStages * kCodeBytes;
  static constexpr int kScales = kCodeScales + kCodeStages * kRows * 4;  // [ring][K 128 | V 128] fp32
  static constexpr int kMl = kScales + (Q8 ? kScaleRing * 2 * kRows * 4 : 0);  // [128] (maximum, sum)
  static constexpr int kRedo = kMl + kRows * 8;                    // 32 words and one
  static constexpr int kBars = kRedo + 256;
  static constexpr int kSmem = kBars + 512 + 1024;
  static_assert(kSmem <= 232448 - 64, "shared memory");
  static constexpr int kThreads = Q8 ? 512 : 384;
  // registers: a block of 384 threads starts with 168 each, one of 512 with 128; the warpgroups' shares add up to that
  static constexpr int kSoftRegs = Q8 ? 168 : 208;
  static constexpr int kOtherRegs = Q8 ? 88 : 88;
  static_assert(2 * kSoftRegs + (kThreads / 128 - 2) * kOtherRegs <= (kThreads / 128) * (Q8 ? 128 : 168), "registers");
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
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
               "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
               "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

// 16 rows at a time, laid out as a product's fragments: lane holds columns 8 g + 2 (lane & 3) and the next one of rows
// lane / 4 (words 4 g, 4 g + 1) and lane / 4 + 8 (words 4 g + 2, 4 g + 3).
__device__ __forceinline__ void tmem_ld_frag128(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12,"
               "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32,"
               "%33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52,"
               "%53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                 "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                 "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                 "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
                 "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]),
                 "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
                 "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
                 "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_frag32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13,"
               "%14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_frag32(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11,"
               "%12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
                 "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15]), "r"(taddr));
}
// The same of 16-bit pairs: word 2 g holds columns 8 g + 2 (lane & 3) and the next one of row lane / 4, 2 g + 1 of lane / 4 + 8.
__device__ __forceinline__ void tmem_st_pairs32(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr));
}

// One lane of a converged warp. The compiler knows that elect.sync leaves a single thread, and issues a tensor-core
// product, a commit or a TMA copy in its branch once; behind `lane == 0` it has to allow for several threads, which
// measured 91 cycles a product (64 is the hardware's rate) and 60 a commit (7).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// mbar_wait with its polls in one asm loop: 43 cycles where the phase is already over, 179 as a C++ loop.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, int where) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, %3;\n\t"
      "POLL:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "sub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra POLL;\n\t"
      "DONE:\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "n"(MG_SPIN_LIMIT)
      : "memory");
  if (!ok) mg_record_error(MG_ERR_TIMEOUT, where);
  return ok != 0;
}

// tcgen05.wait::ld that the loaded registers pass through: nothing that uses them can be moved ahead of it.
__device__ __forceinline__ void wait_ld8(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}

template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Pairs of fp32 in one 64-bit register: one FMA-pipe instruction for two values.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

struct RagArgs {
  int64_t rows, max_rows, num_blocks;
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
  int *err_code, *err_info;
};

// A CTA's k-th piece of work: an entry of the list and a K/V head. The list is sorted, longest first, and dealt out
// forwards and backwards in turn, which evens out the CTAs' sums.
struct RagWork {
  RagItem it;
  int head, tiles;    // K/V head; K/V tiles of the item
  int n0, n1;         // K/V tiles that each softmax warpgroup visits
  bool dual;          // one row tile: the warpgroups take its K/V tiles in turn
};

__device__ __forceinline__ int rag_index(int k, int total) {
  const int g = (int)gridDim.x, c = (int)blockIdx.x;
  const int64_t i = (int64_t)k * g + (k & 1 ? g - 1 - c : c);
  return i < total ? (int)i : -1;
}
__device__ __forceinline__ RagItem rag_item(const RagArgs& p, int index) {
  RagItem r = {};
  if (index >= 0) {
    const int4* src = reinterpret_cast<const int4*>(p.work + p.list_off) + 2 * (index / p.hkv);
    const int4 a = __ldg(src), b = __ldg(src + 1);
    r.seq = a.x, r.row0 = a.y, r.n_tok = a.z, r.pos0 = a.w;
    r.kt0 = b.x, r.kt1 = b.y, r.slot = b.z, r.kv_len = b.w;
  }
  return r;
}
// A CTA's way through its work: all of it, and (again) the pieces that have to be done over.
constexpr int kRedoWords = 32;
struct RagWalk {
  int k, total, index;
  RagItem it;
  __device__ __forceinline__ void start(const RagArgs& p, int n, const volatile uint32_t* redo) {
    k = -1;
    total = n;
    next(p, redo);
  }
  // redo: the pieces to do over, one bit each (the last bit stands for all behind it too), or null
  __device__ __forceinline__ void next(const RagArgs& p, const volatile uint32_t* redo) {
    do {
      index = rag_index(++k, total);
    } while (redo && index >= 0 && !(redo[min(k >> 5, kRedoWords - 1)] >> (k < 32 * kRedoWords ? k & 31 : 31) & 1u));
    it = rag_item(p, index);
  }
};
// The work of an item; one that does not fit this call's arrays (fewer rows than the plan has) has no tiles.
__device__ __forceinline__ RagWork rag_work(const RagArgs& p, const RagItem& it, int index) {
  RagWork w;
  w.it = it;
  w.head = index % p.hkv;
  const bool fits = it.row0 >= 0 && it.n_tok > 0 && (int64_t)it.row0 + it.n_tok <= p.rows && it.seq >= 0 && it.seq < p.b &&
                    it.kt0 >= 0 && it.kt1 > it.kt0 && (int64_t)it.kv_len <= (int64_t)p.max_blocks * 16 &&
                    (int64_t)(it.kt1 - 1) * kRows < it.kv_len && it.slot < p.max_slots;
  if (!fits) {
    w.it.n_tok = 0;
    w.n0 = w.n1 = w.tiles = 0;
    w.dual = false;
    return w;
  }
  const int tiles = it.kt1 - it.kt0;
  w.dual = it.n_tok <= p.tok_tile;
  if (w.dual) {
    w.n0 = (tiles + 1) >> 1;
    w.n1 = tiles >> 1;
    w.tiles = tiles;
  } else {  // the first row tile ends at its own last token
    const int last = it.pos0 + p.tok_tile - 1;
    w.n0 = max(0, min(it.kt1, last / kRows + 1) - it.kt0);
    w.n1 = tiles;
    w.tiles = tiles;
  }
  return w;
}

// Whether rows [r0, r1) of a V tile hold an infinity or a NaN (by the warps of a warpgroup, t = 0 .. 127; the answer is the
// warp's). A bf16 infinity or NaN has all exponent bits set: adding one at the lowest of them carries out.
template <int D>
__device__ __noinline__ bool odd_rows(const uint8_t* v, int r0, int r1, int t) {
  constexpr int kChunks = D / 8;
  uint32_t acc = 0;
  for (int x = r0 * kChunks + t; x < r1 * kChunks; x += 128) {
    const uint4 q = *reinterpret_cast<const uint4*>(v + chunk_at<D>(x / kChunks, x % kChunks));
    acc |= ((q.x & 0x7f807f80u) + 0x00800080u) | ((q.y & 0x7f807f80u) + 0x00800080u) |
           ((q.z & 0x7f807f80u) + 0x00800080u) | ((q.w & 0x7f807f80u) + 0x00800080u);
  }
  return __any_sync(0xffffffffu, (acc & 0x80008000u) != 0);
}

// O += P V over the keys 0 .. see of a tile that the thread's row sees, from the stage, in the tensor cores' place. ts, to:
// the warp's tensor-memory addresses of P and O; `more`: something is in O already. (Not inlined, like odd_rows: in the
// loop's body their registers and code cost every call 5 % and serve none but those with an infinity or NaN in V.)
template <int D>
__device__ __noinline__ void values_by_hand(const uint8_t* v, uint32_t ts, uint32_t to, int see, bool more) {
#pragma unroll 1
  for (int c = 0; c < D; c += 8) {
    float o[8] = {};
    uint32_t x8[8];
    if (more) {
      tmem_ld8(to + c, x8);
      wait_ld8(x8);
#pragma unroll
      for (int x = 0; x < 8; ++x) o[x] = __uint_as_float(x8[x]);
    }
#pragma unroll 1
    for (int q = 0; q < kRows; q += 16) {
      uint32_t pr[8];
      tmem_ld8(ts + q / 2, pr);
      wait_ld8(pr);
#pragma unroll
      for (int y = 0; y < 16; ++y) {
        const float pv = y & 1 ? bf16hi(pr[y / 2]) : bf16lo(pr[y / 2]);
        if (q + y <= see) {
          const uint4 x4 = *reinterpret_cast<const uint4*>(v + chunk_at<D>(q + y, c / 8));
          const uint32_t e[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            o[2 * x] = fmaf(pv, bf16lo(e[x]), o[2 * x]);
            o[2 * x + 1] = fmaf(pv, bf16hi(e[x]), o[2 * x + 1]);
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) x8[x] = __float_as_uint(o[x]);
    tmem_st8(to + c, x8);
  }
  tc_wait_st();
}

template <int D, bool Q8>
__global__ void __launch_bounds__(RagCfg<D, Q8>::kThreads, 1)
    ragged_attn_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const RagArgs p) {
  using C = RagCfg<D, Q8>;
  constexpr int NS = C::kStages;
  constexpr int NC = C::kCodeStages > 0 ? C::kCodeStages : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* empty = full + NS;
  uint64_t* cfull = empty + NS;    // [NC] codes landed
  uint64_t* cempty = cfull + NC;   // [NC] codes converted
  uint64_t* qfull = cempty + NC;   // [2] a row tile's Q is in shared memory
  uint64_t* qfree = qfull + 2;     // [2] its products are done
  uint64_t* sfull = qfree + 2;     // [2] scores are in tensor memory (and the warpgroup's earlier P V is done)
  uint64_t* pready = sfull + 2;    // [2] probabilities are
  uint64_t* ofull = pready + 2;    // [2] the item's output is complete
  uint64_t* looked = ofull + 2;    // [2] every warp has looked over a masked tile's V rows (second pass)
  uint64_t* mlready = looked + 2;  // the second warpgroup's (maximum, sum) are in shared memory
  uint64_t* merged = mlready + 1;  // ... and its output has been read
  uint64_t* drained = merged + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* skip = reinterpret_cast<volatile int*>(tmem_holder + 1);  // [2] the softmax threads did a tile's P V
  // [2] the last piece (its place in the CTA's list, from 1) with an infinity or NaN among V rows that some row may not
  // see. The warps of a warpgroup enter a piece at times of their own, so a flag that one of them cleared there could wipe
  // out what another has found already; a finding's own name needs no clearing.
  volatile int* odd_v = skip + 2;
  volatile uint32_t* redo = reinterpret_cast<volatile uint32_t*>(smem + C::kRedo);  // pieces for a second pass ...
  volatile uint32_t* redo_any = redo + kRedoWords;                                   // ... and whether there are any
  auto block_barrier = [] { asm volatile("bar.sync 1, %0;" ::"n"(C::kThreads) : "memory"); };

  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x <= kRedoWords) redo[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    mg_set_error_words(p.err_code, p.err_info);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], Q8 ? 4 : 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < NC; ++s) {
      mbar_init(&cfull[s], 1);
      mbar_init(&cempty[s], 4);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&qfull[w], 1);
      mbar_init(&qfree[w], 1);
      mbar_init(&sfull[w], 1);
      mbar_init(&pready[w], 4);
      mbar_init(&ofull[w], 1);
      mbar_init(&looked[w], 4);
      skip[w] = 0;
      odd_v[w] = 0;
    }
    mbar_init(mlready, 4);
    mbar_init(merged, 4);
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
  const uint32_t tmem = 0;  // the CTA holds all of tensor memory
  griddep_wait();
  const RagHead head = *reinterpret_cast<const RagHead*>(p.work);
  const bool planned = rag_made_for(head, p.max_rows, p.b, p.hq, p.hkv, p.max_blocks);
  const int total = planned ? head.n_list * p.hkv : 0;  // (the merge records it)

  if (warp >= 8) {
    regs_dec<C::kOtherRegs>();
    bool ok = true;
    RagWalk walk;
    if (warp == 8) {
      // ---------------- tensor-core issue ----------------
      const uint32_t sq = smem_u32(smem), sr = smem_u32(smem + C::kRing);
      const uint64_t q_desc = rag_desc<D>(sq, 16), k_desc = rag_desc<D>(sr, 16), v_desc = rag_desc<D>(sr, C::kSlabBytes);
      int base = 0;
      uint32_t pp = 0, pq = 0;  // phase bits of pready and qfull, one per row tile
      for (int pass = 0; pass < 2; ++pass) {
        walk.start(p, total, pass ? redo : nullptr);
        while (walk.index >= 0 && ok) {
          const RagWork wk = rag_work(p, walk.it, walk.index);
          walk.next(p, pass ? redo : nullptr);
          const int tiles = uniform(wk.tiles), n0 = uniform(wk.n0), n1 = uniform(wk.n1);
          const bool dual = uniform(wk.dual) != 0;
          // S_w = Q_w K_j^T (in a branch of one thread)
          auto scores = [&](int w, int j) {
            const uint64_t a = q_desc + (uint64_t)(w * (C::kTileBytes >> 4));
            const uint64_t b = k_desc + (uint64_t)(((base + 2 * j) % NS) * (C::kTileBytes >> 4));
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
              const uint64_t off = (uint64_t)(((x * 32 / C::kSlab) * C::kSlabBytes + (x * 32) % C::kSlab) >> 4);
              tc_mma_ss((uint32_t)(w * kRows), a + off, b + off, C::kIdescS, x > 0);
            }
            tc_commit(&sfull[w]);
          };
          auto await_k = [&](int j) {
            const int i = base + 2 * j;
            ok = ok && bar_wait(&full[i % NS], (i / NS) & 1, 515);
            tc_fence_after();
          };
          const int step = dual ? 2 : 1;
#pragma unroll (Q8 ? 1 : 2)
          for (int w = 0; w < 2; ++w) {
            const int n = w ? n1 : n0;
            if (n == 0 || !ok) continue;
            ok = bar_wait(&qfull[w], (pq >> w) & 1, 514);
            pq ^= 1u << w;
            const int j = dual ? w : 0;
            if (dual || w == 0 || n0 == 0) await_k(j);
            if (!ok) break;
            if (elect_one()) {
              scores(w, j);
              if (n == 1) tc_commit(&qfree[w]);
              if (dual || w == 1) tc_commit(&empty[(base + 2 * j) % NS]);
            }
            __syncwarp();
          }
          for (int j = 0; j < tiles && ok; ++j) {
            const int iv = base + 2 * j + 1, jn = j + step;
            const uint64_t v = v_desc + (uint64_t)((iv % NS) * (C::kTileBytes >> 4));
            ok = bar_wait(&full[iv % NS], (iv / NS) & 1, 516);
            bool k_here = false;
#pragma unroll (Q8 ? 1 : 2)  // (int8: the less code the better, see above)
            for (int w = 0; w < 2; ++w) {
              const int last = dual ? tiles : (w ? n1 : n0);
              if (!ok || (dual ? w != (j & 1) : j >= last)) continue;
              ok = bar_wait(&pready[w], (pp >> w) & 1, 517);
              if (!ok) break;
              pp ^= 1u << w;
              tc_fence_after();
              const bool by_hand = !Q8 && pass && uniform(skip[w]) != 0;
              if (elect_one()) {
                if (!by_hand) {
                  const uint32_t more = j >= step;  // something is in O already
#pragma unroll
                  for (int x = 0; x < kRows / 16; ++x)  // 16 keys a step: 16 rows of V
                    tc_mma_ts(C::kO + (uint32_t)(w * D), (uint32_t)(w * kRows + x * 8),
                              v + (uint64_t)((x * 16 * C::kSlab) >> 4), C::kIdescO, x > 0 ? 1u : more);
                }
                if (dual || w == 1) tc_commit(&empty[iv % NS]);
                if (jn >= last) tc_commit(&ofull[w]);
              }
              __syncwarp();
              if (jn < last) {
                if (!k_here) await_k(jn);
                k_here = true;
                if (!ok) break;
                if (elect_one()) {
                  scores(w, jn);
                  if (jn + step >= last) tc_commit(&qfree[w]);
                  if (dual || w == 1) tc_commit(&empty[(base + 2 * jn) % NS]);
                }
                __syncwarp();
              }
            }
          }
          base += 2 * tiles;
        }
        if (Q8 || pass) break;
        block_barrier();
        if (!*redo_any) break;
      }
      if (elect_one()) tc_commit(drained);
      __syncwarp();
      bar_wait(drained, 0, 519);
    } else if (warp == 9 || warp == 11) {
      // ---------------- K/V loads: K_0, V_0, K_1, V_1, ..., K by one warp and V by another ----------------
      // bf16: a TMA copy for each block and slab; int8: bulk copies of a block's codes and scales. Lane b < 8 holds the
      // tile's b-th block id, fetched a tile ahead; one lane starts the copies. (Where the ring is of odd length, a stage's
      // loads alternate between the warps. None can take an older release of a stage for the one it waits for: releases
      // come nearly in the order of the loads, and its own last wait was for a later one than that.)
      const int kv = warp == 11;
      int i = kv;  // the next load's place in that order
      const int blk = lane & 7;
      for (int pass = 0; pass < 2; ++pass) {
        walk.start(p, total, pass ? redo : nullptr);
        while (walk.index >= 0 && ok) {
          const RagWork wk = rag_work(p, walk.it, walk.index);
          if (wk.it.n_tok == 0) mg_record_error(MG_ERR_DEVICE, 510);
          walk.next(p, pass ? redo : nullptr);
          const int32_t* table = p.tables + (int64_t)wk.it.seq * p.max_blocks;
          const int blocks = (wk.it.kv_len + 15) >> 4;
          int b0 = wk.it.kt0 * 8;
          int32_t id_next = wk.tiles > 0 && b0 + blk < blocks ? table[b0 + blk] : 0;
          for (int j = 0; j < wk.tiles && ok; ++j, b0 += 8, i += 2) {
            const int nb = min(8, blocks - b0);
            const int32_t id = id_next;
            const bool good = id >= 0 && id < p.num_blocks;
            if (blk < nb && !good) mg_record_error(MG_ERR_DEVICE, 511);
            if (b0 + 8 + blk < blocks) id_next = table[b0 + 8 + blk];
            if constexpr (Q8) {
              const int s = i % NC;
              if (i >= NC) ok = ok && bar_wait(&cempty[s], ((i / NC) - 1) & 1, 512);
              if (!ok) break;
              // a block that is not in the pool is read as the pool's first (its error has been recorded)
              const int row = (good ? id : 0) * p.hkv + wk.head;
              if (elect_one()) mbar_arrive_expect_tx(&cfull[s], (uint32_t)(nb * 16 * (D + 4)));
#pragma unroll 1
              for (int y = 0; y < 8; ++y) {
                const int64_t r = (int64_t)__shfl_sync(0xffffffffu, row, y) * 16;
                if (y < nb && elect_one()) {
                  bulk_load_smem(smem + C::kCodes + s * C::kCodeBytes + y * 16 * D, (kv ? p.v8 : p.k8) + r * D, 16 * D,
                                 &cfull[s]);
                  bulk_load_smem(smem + C::kCodeScales + s * kRows * 4 + y * 64, (kv ? p.vs : p.ks) + r, 64, &cfull[s]);
                }
                __syncwarp();
              }
            } else {
              const int s = i % NS;
              if (i >= NS) ok = ok && bar_wait(&empty[s], ((i / NS) - 1) & 1, 512);
              if (!ok) break;
              // (a block that is not in the pool is read behind its end: as zeros)
              const int row = (int)(good ? (id * p.hkv + wk.head) * 16 : p.num_blocks * p.hkv * 16);
              if (elect_one()) mbar_arrive_expect_tx(&full[s], (uint32_t)(nb * 16 * D * 2));
#pragma unroll
              for (int y = 0; y < 8; ++y) {
                const int r = __shfl_sync(0xffffffffu, row, y);
                if (y < nb && elect_one()) {
#pragma unroll
                  for (int x = 0; x < C::kSlabs; ++x)
                    tma_load_2d(smem + C::kRing + s * C::kTileBytes + x * C::kSlabBytes + y * 16 * C::kSlab, kv ? &tv : &tk,
                                &full[s], x * (C::kSlab / 2), r);
                }
                __syncwarp();
              }
            }
          }
        }
        if (Q8 || pass) break;
        block_barrier();
        if (!*redo_any) break;
      }
      // the loads that were started have landed before this CTA's memory goes to another
      const int all = i - kv;
      if constexpr (Q8) {
        for (int x = max(0, all - NC); x < all; ++x)
          if ((x & 1) == kv) bar_wait(&cfull[x % NC], (x / NC) & 1, 513);
      } else {
        for (int x = max(0, all - NS); x < all; ++x)
          if ((x & 1) == kv) bar_wait(&full[x % NS], (x / NS) & 1, 513);
      }
    } else if (warp == 10) {
      // ---------------- Q loads: a row tile's tokens x heads of the group, as soon as the products before are done ------
      int c0 = 0, c1 = 0;  // loads so far
      for (int pass = 0; pass < 2; ++pass) {
        walk.start(p, total, pass ? redo : nullptr);
        while (walk.index >= 0 && ok) {
          const RagWork wk = rag_work(p, walk.it, walk.index);
          walk.next(p, pass ? redo : nullptr);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            int& c = w ? c1 : c0;
            if ((w ? wk.n1 : wk.n0) == 0 || !ok) continue;
            if (c > 0) ok = bar_wait(&qfree[w], (c - 1) & 1, 524);
            if (!ok) break;
            ++c;
            if (elect_one()) {
              mbar_arrive_expect_tx(&qfull[w], (uint32_t)(C::kSlabs * p.tok_tile * p.group * C::kSlab));
#pragma unroll
              for (int s = 0; s < C::kSlabs; ++s)
                tma_load_3d(smem + w * C::kTileBytes + s * C::kSlabBytes, &tq, &qfull[w], s * (C::kSlab / 2),
                            wk.head * p.group, wk.it.row0 + (wk.dual ? 0 : w * p.tok_tile));
            }
            __syncwarp();
          }
        }
        if (Q8 || pass) break;
        block_barrier();
        if (!*redo_any) break;
      }
      if (c0 > 0) bar_wait(&qfull[0], (c0 - 1) & 1, 525);
      if (c1 > 0) bar_wait(&qfull[1], (c1 - 1) & 1, 525);
    } else if (Q8 && warp >= 12) {
      // ---------------- int8 codes -> bf16 tiles, swizzled ----------------
      const int t = threadIdx.x - 12 * 32;
      float* scales = reinterpret_cast<float*>(smem + C::kScales);
      constexpr int kParts = D / 16;              // 16-byte pieces of a vector of codes
      constexpr int kPer = kRows * kParts / 128;  // pieces per thread and tile
      int i = 0, tile = 0;
      for (int pass = 0; pass < 2; ++pass) {
        walk.start(p, total, pass ? redo : nullptr);
        while (walk.index >= 0 && ok) {
          const RagWork wk = rag_work(p, walk.it, walk.index);
          walk.next(p, pass ? redo : nullptr);
          for (int j = 0; j < wk.tiles && ok; ++j, ++tile) {
            const int keys = wk.it.kv_len - (wk.it.kt0 + j) * kRows;  // of the tile, where fewer than 128
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv, ++i) {
              const int s = i % NS, sc = i % NC;
              ok = ok && bar_wait(&cfull[sc], (i / NC) & 1, 526);
              if (i >= NS) ok = ok && bar_wait(&empty[s], ((i / NS) - 1) & 1, 527);
              if (!ok) break;
              const uint8_t* src = smem + C::kCodes + sc * C::kCodeBytes;
              uint8_t* dst = smem + C::kRing + s * C::kTileBytes;
              // (a batch's loads before its stores: the compiler cannot tell the two buffers apart; and few batches unrolled,
              // for the instruction caches)
              const float scale = reinterpret_cast<const float*>(smem + C::kCodeScales)[sc * kRows + t];
              constexpr int kBatch = kPer < 2 ? kPer : 2;
#pragma unroll 1
              for (int x0 = 0; x0 < kPer; x0 += kBatch) {
                uint4 c[kBatch];
#pragma unroll
                for (int x = 0; x < kBatch; ++x) c[x] = *reinterpret_cast<const uint4*>(src + ((x0 + x) * 128 + t) * 16);
#pragma unroll
                for (int x = 0; x < kBatch; ++x) {
                  const int piece = (x0 + x) * 128 + t, r = piece / kParts, q = (piece % kParts) * 2;
                  if (r >= keys) c[x] = make_uint4(0, 0, 0, 0);
                  uint4 lo, hi;
                  i8x4_to_bf16x4(c[x].x, lo.x, lo.y);
                  i8x4_to_bf16x4(c[x].y, lo.z, lo.w);
                  i8x4_to_bf16x4(c[x].z, hi.x, hi.y);
                  i8x4_to_bf16x4(c[x].w, hi.z, hi.w);
                  // (a row's second 128 bytes lie on the banks of its first: those threads store the other way round)
                  const int swap = (q >> 3) & 1;
                  *reinterpret_cast<uint4*>(dst + chunk_at<D>(r, q + swap)) = swap ? hi : lo;
                  *reinterpret_cast<uint4*>(dst + chunk_at<D>(r, q + 1 - swap)) = swap ? lo : hi;
                }
              }
              scales[(tile % C::kScaleRing) * 2 * kRows + kv * kRows + t] =
                  t < keys ? scale : 0.f;
              fence_async_smem();
              __syncwarp();
              if (lane == 0) {
                mbar_arrive(&cempty[sc]);
                mbar_arrive(&full[s]);
              }
            }
          }
        }
        if (Q8 || pass) break;
        block_barrier();
        if (!*redo_any) break;
      }
    }
  } else {
    // ---------------- softmax: one thread per row ----------------
    regs_inc<C::kSoftRegs>();
    const int w = warp >> 2, t = threadIdx.x & 127;  // warpgroup, row
    const int my_tok = t / p.group;
    const int64_t row_stride = (int64_t)p.hq * D;
    const int64_t my_off = (int64_t)my_tok * row_stride + (t % p.group) * D;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lane_base + (uint32_t)(w * kRows), to = tmem + lane_base + C::kO + (uint32_t)(w * D);
    const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
    constexpr int kR = Q8 ? 4 : 1;  // rows whose maximum and sum the thread holds: t, or as fragments lane / 4 + 8 k
    [[maybe_unused]] int frag_tok[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) frag_tok[k] = ((t & ~31) + (lane >> 2) + 8 * k) / p.group;
    bool ok = true;
    int base = 0, cs = 0, co = 0, looks = 0, duals = 0, tile0 = 0;
    RagWalk walk;
    // (a function of its own for the second pass: what only that does would cost the first one registers, 5 % of its time)
    auto softmax_pass = [&](auto again_tag) {
      constexpr bool kAgain = decltype(again_tag)::value;
      walk.start(p, total, kAgain ? redo : nullptr);
      while (walk.index >= 0 && ok) {
        const RagWork wk = rag_work(p, walk.it, walk.index);
        const int piece = walk.k;
        walk.next(p, kAgain ? redo : nullptr);
        const RagItem& it = wk.it;
        const int tok0 = wk.dual ? 0 : w * p.tok_tile;
        const int valid = max(0, min(p.tok_tile, it.n_tok - tok0)) * p.group;
        const int first_pos = it.pos0 + tok0, my_pos = first_pos + my_tok;
        const bool warp_on = (warp & 3) * 32 < valid;
        const int n = w ? wk.n1 : wk.n0;
        float mr[kR];     // the maxima in use of the thread's rows, in score units
        uint64_t lr[kR];  // the sums, in two halves
#pragma unroll
        for (int k = 0; k < kR; ++k) {
          mr[k] = -INFINITY;
          lr[k] = 0;
        }
        for (int i = 0; i < n && ok; ++i) {
          const int j = wk.dual ? 2 * i + w : i;
          const int key0 = (it.kt0 + j) * kRows;
          ok = bar_wait(&sfull[w], cs++ & 1, 520);
          if (!ok) break;
          tc_fence_after();
          const bool masked = key0 + kRows - 1 > first_pos;  // some row of the tile does not see all its keys
          bool by_hand = false;
          if constexpr (Q8) {  // the values' scales come with V
            const int iv = base + 2 * j + 1;
            ok = bar_wait(&full[iv % NS], (iv / NS) & 1, 521);
            if (!ok) break;
          } else {
            const int iv = base + 2 * j + 1, sv = iv % NS;
            const int r_end = it.kv_len - key0;  // V rows from here on are behind the item's keys
            if (masked && (r_end < kRows || kAgain)) {
              ok = bar_wait(&full[sv], (iv / NS) & 1, 521);
              if (!ok) break;
              uint8_t* v = smem + C::kRing + sv * C::kTileBytes;
              constexpr int kChunks = D / 8;
              for (int x = r_end * kChunks + t; x < kRows * kChunks; x += 128)
                *reinterpret_cast<uint4*>(v + chunk_at<D>(x / kChunks, x % kChunks)) = make_uint4(0, 0, 0, 0);
              fence_async_smem();
              if constexpr (kAgain) {
                const bool odd = odd_rows<D>(v, max(0, first_pos + 1 - key0), min(r_end, kRows), t);
                // (any thread's finding is every thread's; once found it holds for the piece's later tiles too)
                if (lane == 0) {
                  if (odd) odd_v[w] = piece + 1;
                  mbar_arrive(&looked[w]);
                }
                ok = bar_wait(&looked[w], looks & 1, 523);
                ++looks;
                if (!ok) break;
                by_hand = odd_v[w] == piece + 1;
              }
            }
          }
          if (warp_on) {
            if constexpr (Q8) {
              // The scales are one per key and the same for every row: with a row per thread, each would read all of
              // them, and hold 128 scores besides. As fragments a thread has four rows of 32 keys, and works on two of
              // them at a time; four lanes share a row's maximum and sum.
              const uint64_t* sc = reinterpret_cast<const uint64_t*>(
                  reinterpret_cast<const float*>(smem + C::kScales) + ((tile0 + j) % C::kScaleRing) * 2 * kRows) + (lane & 3);
              auto half = [&](uint32_t down, auto masked_tag) {
                constexpr bool kMasked = decltype(masked_tag)::value;
                uint32_t raw[64];
                tmem_ld_frag128(ts + down, raw);
                tc_wait_ld();
                auto at = [&](int k, int g, int e) -> float& {  // row k of the two, key 8 g + 2 (lane & 3) + e
                  return reinterpret_cast<float&>(raw[4 * g + 2 * k + e]);
                };
#pragma unroll
                for (int g = 0; g < 16; ++g) {
                  const uint64_t f = sc[4 * g];
#pragma unroll
                  for (int k = 0; k < 2; ++k) unpair(mul2(pair(at(k, g, 0), at(k, g, 1)), f), at(k, g, 0), at(k, g, 1));
                }
                int see[2];  // keys 8 g + e with 8 g + e <= see are the row's
                bool grow[2];
                float m_new[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  see[k] = first_pos + frag_tok[k] - key0 - 2 * (lane & 3);
                  const float m = mr[k];
                  float a = m, b = m;
#pragma unroll
                  for (int g = 0; g < 16; ++g) {
                    if constexpr (kMasked) {
                      at(k, g, 0) = 8 * g <= see[k] ? at(k, g, 0) : -INFINITY;
                      at(k, g, 1) = 8 * g + 1 <= see[k] ? at(k, g, 1) : -INFINITY;
                    }
                    (g & 1 ? b : a) = max3(g & 1 ? b : a, at(k, g, 0), at(k, g, 1));
                  }
                  a = fmaxf(a, b);
                  a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
                  a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
                  grow[k] = m == -INFINITY || (a - m) * p.scale_log2 > 8.f;
                  m_new[k] = grow[k] ? a : m;
                }
                if (i > 0 && __any_sync(0xffffffffu, grow[0] || grow[1])) {
                  float f[2];
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    const float m = mr[k];
                    f[k] = m == -INFINITY ? 0.f : ex2((m - m_new[k]) * p.scale_log2);
                    lr[k] = mul2(lr[k], pair(f[k], f[k]));
                  }
#pragma unroll 1
                  for (int c = 0; c < D; c += 32) {
                    uint32_t o[16];
                    tmem_ld_frag32(to + down + c, o);
                    tc_wait_ld();
#pragma unroll
                    for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f[(x >> 1) & 1]);
                    tmem_st_frag32(to + down + c, o);
                  }
                }
                uint64_t off2[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  mr[k] = m_new[k];
                  const float off = m_new[k] == -INFINITY ? 0.f : -m_new[k] * p.scale_log2;
                  off2[k] = pair(off, off);
                }
#pragma unroll
                for (int g0 = 0; g0 < 16; g0 += 4) {
                  uint32_t pk[8];
#pragma unroll
                  for (int g = g0; g < g0 + 4; ++g) {
                    const uint64_t f = sc[kRows / 2 + 4 * g];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                      float a, b;
                      unpair(fma2(pair(at(k, g, 0), at(k, g, 1)), scale2, off2[k]), a, b);
                      a = ex2(a);
                      b = ex2(b);
                      lr[k] = add2(lr[k], pair(a, b));
                      unpair(mul2(pair(a, b), f), a, b);
                      if constexpr (kMasked) {  // (nothing of a masked key's scale, whatever it is)
                        a = 8 * g <= see[k] ? a : 0.f;
                        b = 8 * g + 1 <= see[k] ? b : 0.f;
                      }
                      pk[2 * (g - g0) + k] = pack_bf16x2(a, b);
                    }
                  }
                  tmem_st_pairs32(ts + down + g0 * 4, pk);
                }
              };
              // (compiled twice, since tests inside the loops would cut them into pieces too short to schedule; and once for
              // both halves, which take turns in the same registers: unrolled, the code does not stay in the
              // instruction caches)
#pragma unroll 1
              for (int h = 0; h < 2; ++h) {
                if (masked) half((uint32_t)(16 * h) << 16, std::true_type{});
                else half((uint32_t)(16 * h) << 16, std::false_type{});
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const float m = mr[k];
                  const uint64_t l = lr[k];
                  const int tok = frag_tok[k];
                  mr[k] = mr[k + 2], mr[k + 2] = m;
                  lr[k] = lr[k + 2], lr[k + 2] = l;
                  frag_tok[k] = frag_tok[k + 2], frag_tok[k + 2] = tok;
                }
              }
            } else {
              float& m = mr[0];
              uint64_t& l2 = lr[0];
              float s[kRows];
#pragma unroll
              for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
              tc_wait_ld();
              const int see = my_pos - key0;  // keys 0 .. see of the tile are this row's
              if (masked) {
#pragma unroll
                for (int h = 0; h < kRows; h += 32) {
                  if (key0 + h + 31 > first_pos) {
#pragma unroll
                    for (int c = h; c < h + 32; ++c) s[c] = c <= see ? s[c] : -INFINITY;
                  }
                }
              }
              float mx[4] = {m, m, m, m};
#pragma unroll
              for (int c = 0; c < kRows; c += 8) {
#pragma unroll
                for (int x = 0; x < 4; ++x) mx[x] = max3(mx[x], s[c + x], s[c + 4 + x]);
              }
              float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
              const bool grow = m == -INFINITY || (m_new - m) * p.scale_log2 > 8.f;
              if (!grow) m_new = m;
              if (i > 0 && __any_sync(0xffffffffu, grow)) {
                const float f = m == -INFINITY ? 0.f : ex2((m - m_new) * p.scale_log2);
                l2 = mul2(l2, pair(f, f));
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                  uint32_t o[32];
                  tmem_ld32(to + c, o);
                  tc_wait_ld();
#pragma unroll
                  for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                  tmem_st32(to + c, o);
                }
              }
              m = m_new;
              const float off = m == -INFINITY ? 0.f : -m * p.scale_log2;
              const uint64_t off2 = pair(off, off);
              uint64_t sum[2] = {l2, 0};
#pragma unroll
              for (int h = 0; h < 4; ++h) {
                uint32_t pk[16];
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                  const int e = h * 32 + 2 * c;
                  float a[4];
#pragma unroll
                  for (int y = 0; y < 2; ++y) {
                    const uint64_t x = fma2(pair(s[e + 2 * y], s[e + 2 * y + 1]), scale2, off2);
                    unpair(x, a[2 * y], a[2 * y + 1]);
                    a[2 * y] = ex2(a[2 * y]);
                    a[2 * y + 1] = ex2(a[2 * y + 1]);
                    sum[y] = add2(sum[y], pair(a[2 * y], a[2 * y + 1]));
                  }
                  pk[c] = pack_bf16x2(a[0], a[1]);
                  pk[c + 1] = pack_bf16x2(a[2], a[3]);
                }
                tmem_st16(ts + h * 16, pk);
              }
              l2 = add2(sum[0], sum[1]);
            }
            tc_wait_st();
            if constexpr (kAgain) {
              if (by_hand) {
                values_by_hand<D>(smem + C::kRing + ((base + 2 * j + 1) % NS) * C::kTileBytes, ts, to, my_pos - key0, i > 0);
              }
            }
          }
          if (kAgain && t == 0) skip[w] = by_hand;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pready[w]);
        }
        base += 2 * wk.tiles;
        tile0 += wk.tiles;
        if (!ok) break;
        // ---------------- epilogue ----------------
        float l = 0.f, ml = -INFINITY;  // of row t
#pragma unroll
        for (int k = 0; k < kR; ++k) {
          float a, b, m = mr[k];
          unpair(lr[k], a, b);
          a += b;
          if constexpr (Q8) {  // from the fragments' rows
            a += __shfl_xor_sync(0xffffffffu, a, 1);
            a += __shfl_xor_sync(0xffffffffu, a, 2);
            a = __shfl_sync(0xffffffffu, a, (lane & 7) * 4);
            m = __shfl_sync(0xffffffffu, m, (lane & 7) * 4);
          }
          if (!Q8 || k == lane >> 3) {
            l = a;
            ml = fmaf(l, 0.f, m * p.scale_log2);  // (a maximum skips NaN, the sum does not: NaN where the row met one)
          }
        }
        const bool both = wk.dual && wk.n1 > 0;  // two states of the same rows: the first warpgroup merges them
        float2* mls = reinterpret_cast<float2*>(smem + C::kMl);
        if (both && w == 1) {
          mls[t] = make_float2(ml, l);
          ok = bar_wait(&ofull[1], co++ & 1, 522);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(mlready);
          ok = ok && bar_wait(merged, duals++ & 1, 528);
          if (!ok) break;
          tc_fence_after();
          continue;
        }
        if (n == 0) {  // a part of a split item whose keys lie behind all of the first row tile's: an empty state
          if (it.slot >= 0 && t < valid)
            p.ws_ml[((int64_t)it.slot * p.hkv + wk.head) * (2 * kRows) + w * kRows + t] = make_float2(-INFINITY, 0.f);
          continue;
        }
        ok = bar_wait(&ofull[w], co++ & 1, 522);
        float f0 = 1.f, f1 = 0.f;
        // a state whose row saw no key there is left out of a merge, whatever its output holds; one whose weight is merely
        // nothing in 32 bits is not, for an infinity or NaN in it counts
        bool out0 = false, out1 = true;
        if (both) {
          ok = ok && bar_wait(mlready, duals++ & 1, 529);
          const float2 o1 = mls[t];
          const float top = fmaxf(ml, o1.x);
          f0 = ml == -INFINITY ? 0.f : exp2f(ml - top);
          f1 = o1.x == -INFINITY ? 0.f : exp2f(o1.x - top);
          l = (f0 == 0.f ? 0.f : f0 * l) + (f1 == 0.f ? 0.f : f1 * o1.y);
          out0 = ml == -INFINITY && top != -INFINITY;
          out1 = o1.x == -INFINITY && top != -INFINITY;
          ml = fmaf(l, 0.f, top);  // (NaN beside an empty state too: fmaxf has skipped it)
        }
        if (!ok) break;
        tc_fence_after();
        if (warp_on) {
          float odd_sum = 0.f;  // a NaN once a value is one, or an infinity
          // (every row sees a key: no sum at all means that all its scores were -inf; its output, 0 / 0, is NaN)
          const float inv = it.slot >= 0 ? 1.f : 1.f / l;
          f0 *= inv;
          f1 *= inv;
          const int64_t slot_row = ((int64_t)it.slot * p.hkv + wk.head) * (2 * kRows) + (wk.dual ? 0 : w * kRows) + t;
          __nv_bfloat16* dst = p.out + (int64_t)(it.row0 + tok0) * row_stride + (int64_t)wk.head * p.group * D + my_off;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(to + c, o);
            tc_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = out0 ? 0u : __float_as_uint(__uint_as_float(o[x]) * f0);
            if (both) {
              uint32_t o1[32];
              tmem_ld32(to + D + c, o1);
              tc_wait_ld();
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (!out1) o[x] = __float_as_uint(fmaf(__uint_as_float(o1[x]), f1, __uint_as_float(o[x])));
            }
            if constexpr (!Q8) {
#pragma unroll
              for (int x = 0; x < 32; ++x) odd_sum = fmaf(__uint_as_float(o[x]), 0.f, odd_sum);
            }
            if (t < valid) {
              if (it.slot < 0) {
#pragma unroll
                for (int x = 0; x < 32; x += 8)
                  *reinterpret_cast<uint4*>(dst + c + x) =
                      make_uint4(pack_bf16x2(__uint_as_float(o[x]), __uint_as_float(o[x + 1])),
                                 pack_bf16x2(__uint_as_float(o[x + 2]), __uint_as_float(o[x + 3])),
                                 pack_bf16x2(__uint_as_float(o[x + 4]), __uint_as_float(o[x + 5])),
                                 pack_bf16x2(__uint_as_float(o[x + 6]), __uint_as_float(o[x + 7])));
              } else {
#pragma unroll
                for (int x = 0; x < 32; x += 4)
                  *reinterpret_cast<uint4*>(p.ws_o + slot_row * D + c + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
              }
            }
          }
          if (it.slot >= 0 && t < valid) p.ws_ml[slot_row] = make_float2(ml, l);
          if (!Q8 && !kAgain && t < valid && odd_sum != 0.f) {
            // Zero times an infinite or NaN value of a masked key may be in there: the piece is done over with a look at V.
            atomicOr(const_cast<uint32_t*>(redo + min(piece >> 5, kRedoWords - 1)),
                     1u << (piece < 32 * kRedoWords ? piece & 31 : 31));
            *redo_any = 1;
          }
        }
        tc_fence_before();
        if (both) {
          __syncwarp();
          if (lane == 0) mbar_arrive(merged);
        }
      }
    };
    softmax_pass(std::false_type{});
    if constexpr (!Q8) {
      block_barrier();
      if (*redo_any) softmax_pass(std::true_type{});
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(*tmem_holder, 512);
  }
}

// Merge of the partial states of the items that were split: row r of item m, in slot order,
//   M = max m_s,  out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.
// A warp takes a row of one K/V head, D / 32 columns per lane. Bound by latency (a chain of the plan's head, the items'
// table, states and outputs): so the rows of all items are dealt out evenly over as many warps as the machine holds, and
// the first batch of outputs is fetched while the states are.
// Measured (attention and merge): 16 chunks over up to 3800 cached tokens, 71.5 us with a CTA for every item, head and
// eighth of the rows, 59.6 so; 62 with batches of eight parts, which only a single token over a long cache gains from.
constexpr int kMergeWarps = 8;
constexpr int kMergeBatch = 4;  // parts in flight
constexpr int kMergeCtas = 4;   // CTAs that an SM holds

template <int D>
struct MergeVec { using type = float; };
template <>
struct MergeVec<64> { using type = float2; };
template <>
struct MergeVec<128> { using type = float4; };

template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32, kMergeCtas) ragged_merge_kernel(const RagArgs p) {
  using Vec = typename MergeVec<D>::type;
  constexpr int N = D / 32;
  griddep_wait();
  griddep_launch();  // (after the wait: launched before it, a next attention costs 4 of 65 us where nothing is split)
  const int lane = threadIdx.x & 31;
  const RagMerge* items = reinterpret_cast<const RagMerge*>(p.work + p.merge_off);
  const RagHead head = *reinterpret_cast<const RagHead*>(p.work);
  const bool planned = rag_made_for(head, p.max_rows, p.b, p.hq, p.hkv, p.max_blocks);
  if (!planned && blockIdx.x == 0 && threadIdx.x == 0) {
    mg_set_error_words(p.err_code, p.err_info);
    mg_record_error(MG_ERR_DEVICE, 510);
  }
  const int n_items = planned ? head.n_merge : 0;
  // (32-bit indices of a row's 32 vectors: max_slots * hkv is at most 2 * max(multiprocessors, hkv), below 2^18)
  const int step = p.hkv * (2 * kRows);
  int unit = (int)blockIdx.x * kMergeWarps + (threadIdx.x >> 5);  // the warp's next (item, row, head) ...
  int before = 0;                                                 // ... and those of the items passed so far
  for (int i0 = 0; i0 < n_items; i0 += 32) {
    RagMerge mine = {};
    if (i0 + lane < n_items) mine = items[i0 + lane];
    const bool fits = mine.row0 >= 0 && (int64_t)mine.row0 + mine.n_tok <= p.rows && mine.slot0 >= 0 &&
                      mine.n_tok <= 2 * p.tok_tile && mine.parts > 0 && mine.slot0 + mine.parts <= p.max_slots;
    // (an item of more rows than the call's does not: the attention kernel has recorded it)
    const int units = fits ? mine.n_tok * p.group * p.hkv : 0;
    int upto = units;  // units of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += below;
    }
    const int all = __shfl_sync(0xffffffffu, upto, 31);
    for (; unit < before + all; unit += (int)gridDim.x * kMergeWarps) {
      const int at_unit = unit - before;
      const int owner = __ffs(__ballot_sync(0xffffffffu, upto > at_unit)) - 1;
      const int local = at_unit - __shfl_sync(0xffffffffu, upto - units, owner);
      const int row0 = __shfl_sync(0xffffffffu, mine.row0, owner), slot0 = __shfl_sync(0xffffffffu, mine.slot0, owner);
      const int parts = __shfl_sync(0xffffffffu, mine.parts, owner);
      const int kvh = local % p.hkv, r = local / p.hkv;
      // row r of the item is (token r / group, head r % group); its place in the two tiles
      const int tok = r / p.group, w = tok / p.tok_tile;
      const int first = (slot0 * p.hkv + kvh) * (2 * kRows) + w * kRows + r - w * p.tok_tile * p.group;
      Vec v[kMergeBatch];
      auto fetch = [&](int s) {
        const Vec* src = reinterpret_cast<const Vec*>(p.ws_o) + ((first + s * step) * 32 + lane);
#pragma unroll
        for (int y = 0; y < kMergeBatch; ++y)
          if (s + y < parts) v[y] = src[y * step * 32];
      };
      fetch(0);
      // every lane holds the state of every 32nd part
      float2 ml = lane < parts ? p.ws_ml[first + lane * step] : make_float2(-INFINITY, 0.f);
      float M = ml.x;
      for (int s = lane + 32; s < parts; s += 32) M = fmaxf(M, p.ws_ml[first + s * step].x);
      M = warp_max(M);
      float L = 0.f, f = 0.f, o[N] = {};
      unsigned held = 0;  // the parts that hold a key of the row (the outputs of the others are left out, whatever they are)
#pragma unroll 1
      for (int s = 0; s < parts; s += kMergeBatch) {
        if ((s & 31) == 0) {
          if (s > 0) ml = s + lane < parts ? p.ws_ml[first + (s + lane) * step] : make_float2(-INFINITY, 0.f);
          f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
          L += f == 0.f ? 0.f : f * ml.y;
          held = __ballot_sync(0xffffffffu, ml.x != -INFINITY);
        }
        if (s > 0) fetch(s);
#pragma unroll
        for (int y = 0; y < kMergeBatch; ++y) {
          const float fy = __shfl_sync(0xffffffffu, f, (s + y) & 31);
          if (held >> ((s + y) & 31) & 1u) {
#pragma unroll
            for (int x = 0; x < N; ++x) o[x] = fmaf(fy, reinterpret_cast<const float*>(&v[y])[x], o[x]);
          }
        }
      }
      L = warp_sum(L);
      const float inv = 1.f / L;  // (as in the attention: 0 / 0 where all scores are -inf)
      __nv_bfloat16* dst = p.out + (int64_t)(row0 + tok) * p.hq * D + ((int64_t)kvh * p.group + r % p.group) * D + lane * N;
      if constexpr (N == 4) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
      } else if constexpr (N == 2) {
        *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(o[0] * inv, o[1] * inv);
      } else {
        dst[0] = __float2bfloat16_rn(o[0] * inv);
      }
    }
    before += all;
  }
}

template <int D, bool Q8>
int launch_ragged(const RagArgs& a, const RagShape& s, const void* q, const void* k_pool, const void* v_pool, cudaStream_t st) {
  using C = RagCfg<D, Q8>;
  static bool done[64] = {};
  static std::mutex mu;
  MG_CUDA_TRY(mg_once_per_device(done, mu, [] {
    return cudaFuncSetAttribute(ragged_attn_kernel<D, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  }));
  CUtensorMap tq{}, tk{}, tv{};
  const CUtensorMapSwizzle sw = D >= 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  // Q as [rows][hq][D]: one box is a row tile, tokens times heads of a group, one row of shared memory each
  int rc = mg_make_map_3d(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, q, {(uint64_t)D, (uint64_t)a.hq, (uint64_t)a.rows},
                          {(uint64_t)D * 2, (uint64_t)a.hq * D * 2},
                          {(uint32_t)C::kSlab / 2, (uint32_t)a.group, (uint32_t)a.tok_tile}, sw);
  if (rc) return rc;
  if constexpr (!Q8) {
    const uint64_t rows = (uint64_t)a.num_blocks * a.hkv * 16;
    if (rows > 0x7fffffffull) return MG_ERR_UNSUPPORTED;
    rc = mg_make_map_2d(&tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, k_pool, D, rows, D * 2, C::kSlab / 2, 16, sw);
    if (rc == MG_OK) rc = mg_make_map_2d(&tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, v_pool, D, rows, D * 2, C::kSlab / 2, 16, sw);
    if (rc) return rc;
  }
  const int64_t most = s.max_list * a.hkv;
  if (most > 0x7fffffff || a.hkv > 65535) return MG_ERR_UNSUPPORTED;
  const unsigned ctas = (unsigned)(most < mg_sm_count() ? most : mg_sm_count());
  MG_CUDA_TRY(mg_launch(ragged_attn_kernel<D, Q8>, dim3(ctas), dim3(C::kThreads), C::kSmem, st, 1, tq, tk, tv, a));
  const int64_t merge_rows = (int64_t)s.max_merges * (a.rows < s.tok_item ? a.rows : s.tok_item) * a.hq;
  const int64_t merge_ctas = (merge_rows + kMergeWarps - 1) / kMergeWarps, hold = (int64_t)mg_sm_count() * kMergeCtas;
  MG_CUDA_TRY(mg_launch(ragged_merge_kernel<D>, dim3((unsigned)(merge_ctas < hold ? merge_ctas : hold)),
                        dim3(kMergeWarps * 32), 0, st, 1, a));
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
       reinterpret_cast<uintptr_t>(k_scales) | reinterpret_cast<uintptr_t>(v_scales) | reinterpret_cast<uintptr_t>(work) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return MG_ERR_INVALID_ARG;
  // (an item may be read again after it has been written)
  if (mg_overlap(q, rows * hq * d * 2, out, rows * hq * d * 2)) return MG_ERR_INVALID_ARG;
  RagArgs a{};
  a.rows = rows;
  a.max_rows = max_rows;
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
  const int er = mg_error_words(&a.err_code, &a.err_info);
  if (er) return er;
  cudaStream_t st = mg_stream(stream);
  if (q8) {
    if (d == 32) return launch_ragged<32, true>(a, s, q, k_pool, v_pool, st);
    if (d == 64) return launch_ragged<64, true>(a, s, q, k_pool, v_pool, st);
    return launch_ragged<128, true>(a, s, q, k_pool, v_pool, st);
  }
  if (d == 32) return launch_ragged<32, false>(a, s, q, k_pool, v_pool, st);
  if (d == 64) return launch_ragged<64, false>(a, s, q, k_pool, v_pool, st);
  return launch_ragged<128, false>(a, s, q, k_pool, v_pool, st);
}
