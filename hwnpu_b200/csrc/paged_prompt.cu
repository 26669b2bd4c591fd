// paged_prompt.cu: attention of many new tokens a sequence over a caller's paged 16-bit cache
// (hc_paged_prompt_run) on the 5th-generation tensor cores: softmax(scale Q K^T) V under the causal
// mask, a sliding window and first tokens that stay visible.
//
// Bound. A visible (row, head, slot) costs 4 head_dim flops on the tensor cores and one exponential: with
// head_dim 128 a 128 x 128 tile takes 1,024 clocks of MMA (8,192 flops a clock and SM) and 1,024 of
// the 16 exponentials a clock, with head_dim 64 half the MMA and as many exponentials. Keys and
// values are read from HBM once and from the L2 cache by every CTA.
//
// Rows. The query heads of a kv head share its keys, so a tile's 128 rows are 128 / rep tokens x rep heads
// (row = token * rep + head). A block of rows is two such tiles (A and B), consecutive tokens of one
// sequence: while the softmax of one runs, the tensor cores work for the other.
//
// Slots come in groups of 16 aligned ones, each inside one page, so a tile of 128 slots is one to
// eight TMA boxes (a 64-column half for K), from wherever the pages are: first the groups of the first tokens that stay
// visible, then those from the lowest slot any row of the block sees to its last token. No tile is
// spent on the slots between. Rows of an edge group that no row of the block sees are zeroed in shared
// memory (values only: a hidden score is replaced, but 0 times a hidden NaN would not be 0).
//
// Work. One CTA an SM, or two with head_dim 64. All blocks of all heads and sequences, as many tiles long as they see (and one
// more for a block's start and end), lie one behind the other, and every CTA takes an equal part of that
// line, read from the lengths on the device: ragged sequences, causal triangles and few rows over a
// long cache come out even. A block that a cut falls into is finished by a second kernel, which
// joins the parts' (m, l, O) in order.
//
//   warps 0-3, 4-7  softmax of tile A, B: a thread owns a row. It takes 64 slots (a half of the tile) at
//                   a time: reads the row's scores from tensor memory, keeps the running maximum and
//                   sum in float32, writes P back as 16-bit values over the scores, and at the end O / l
//                   to memory
//   warp 8          copies the groups of K and V (cp.async.bulk.tensor, an mbarrier a ring stage)
//   warps 9, 10     issue the MMAs of tile A, B: S = Q K^T (both operands in shared memory, 128-byte
//                   swizzle), O += P V (P in tensor memory, V in shared memory, MN-major)
//   warp 11         walks the CTA's part of the line, a block ahead of the others, and copies Q
// With head_dim 128 the halves of a tile are two chains (S, softmax, P V, the same half's next S), so that the softmax
// has one half's scores while the tensor cores have the other's P. An MMA of 64 slots takes nearly as long as one
// of 128 (59 clocks against 64), and it still pays: one chain a tile took 565 us for the 16,384-token prompt, two
// 533 then. With 64 there are two CTAs an SM instead.
// The next block's K, V, Q and first scores are under way while a block's last tile and output are.
//
// Arithmetic. S and O are float32. P = exp2(S scale log2(e) - m) is rounded to the cache's type (the MMA
// wants it of V's type); l sums it unrounded in float32. m is moved only when a score passes it by more
// than 2^8, which rescales O in tensor memory; P is at most 256 then, and fp16's P is held 2^7 higher
// so that its smallest weights stand for 2^-32. (A polynomial for some of the exponentials, on the FMA
// pipes, was slower: 617 us against 583 for the 16,384-token prompt with a quarter of them.)
//
// Measured, on several GPUs. 16,384 tokens of 16 heads over 8 of 128, window 4,096: 525 to 537 us, 907 to 927 TFLOP/s
// (56% of a library GEMM's rate); when it took 533, 506 without the copies, 411 without the MMAs, 300 without both and
// the exponentials: no one part bounds it. 512 tokens of 32 heads over 8 after 16,389: 156 to 161 us, 870 to 898
// TFLOP/s, tensor pipe 49%, exponentials 50%. 16 ragged prompts of up to 2,050 of 64 heads over 8 of 64, window 128:
// 177 us, 52% of the issue slots, tensor pipe 12%.
//
// Every mbarrier wait is bounded (about a second of SM clocks): one that runs out records a code that
// hc_device_check reports and lets every other wait of the CTA return; the CTA still waits, bounded,
// for its own copies and MMAs before it frees the tensor memory and exits.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "kernels.h"
#include "paged.h"
#include "tcgen05.cuh"

namespace hc {
namespace {

constexpr int kPpRows = 128;               // rows of a tile (the MMA's M)
constexpr int kPpSlots = 128;              // slots of a tile
constexpr int kPpGroup = 16;               // slots of a group (one TMA box, one K-step of P V)
constexpr int kPpGroups = kPpSlots / kPpGroup;
constexpr int kPpHalfGroups = kPpGroups / 2;  // of a half tile: the step of the softmax
constexpr int kPpSoft = 256;               // threads of the softmax, one a row
constexpr int kPpThreads = kPpSoft + 128;
constexpr int kPpHalf = kPpRows * 128;     // bytes of 128 rows x 64 columns
constexpr float kPpLazy = 8.f;
constexpr float kPpLog2e = 1.4426950408889634f;
constexpr int kPpSegs = 4;                 // blocks the walking warp may be ahead
constexpr int kPpMinPart = 4;              // least tiles of a CTA's part of the line

template <int HD>
struct PpSmem {
  static constexpr int kHalves = HD / 64;
  static constexpr int kTile = kHalves * kPpHalf;  // Q of a tile, or K or V of 128 slots
  // CTAs an SM: tensor memory has room for one with head_dim 128, and for two with 64 when a tile has one half's
  // scores at a time. Four tiles of one chain each then fill each other's gaps, a block's start and end among them:
  // 186 us against 240 with two tiles of two chains for ragged prompts in a window of 128, when both were measured.
  static constexpr int kCtas = HD == 128 ? 1 : 2;
  static constexpr int kBufs = HD == 128 ? 2 : 1;  // halves of S a tile
  static constexpr int kStages = HD == 128 ? 5 : 4;
  static constexpr int kBytes = (2 + kStages) * kTile;  // 224 KB, or 96: 3 KB or 18 a CTA are left
  static constexpr uint32_t kTmem = 2 * (64 * kBufs + HD);  // columns: S_A, S_B, O_A, O_B
  // Scores a thread holds: all 64 of a half, or 32, read twice, where two CTAs leave it 80 registers. One CTA's 168
  // (65,536 / 384) become 208 for the softmax and 88 for the rest, which adds up to the same (2 x 208 + 88 = 3 x 168).
  static constexpr int kHeld = HD == 128 ? 64 : 32;
  static constexpr int kSoftRegs = 208, kRestRegs = 88;
};

__device__ int pp_status_word;  // the first wait that ran out in any launch (0: none)

// tc_wait, and it gives up at once when another wait of the CTA has.
__device__ __forceinline__ void pp_wait(uint64_t *b, unsigned parity, volatile int *dead, int code) {
  if (tc_try(b, parity)) return;
  const long long t0 = clock64();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (tc_try(b, parity)) return;
    if (*dead) return;
    if (clock64() - t0 > kTcSpin) {
      atomicCAS(&pp_status_word, 0, code);
      *dead = 1;
      return;
    }
  }
}

// Shared-memory descriptors with the 128-byte swizzle (8 rows x 128 bytes an atom): K-major (rows are M or
// N, 8-row groups 1,024 bytes apart), and MN-major (rows are K; the next 64 columns lbo further).
__device__ __forceinline__ uint64_t pp_desc(uint32_t saddr, uint32_t lbo) {
  return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(lbo >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor of kind::f16: float32 D, M = 128, N = n, A K-major, B K-major or (vt) MN-major.
__device__ __forceinline__ uint32_t pp_idesc(bool bf16, int n, bool vt) {
  const uint32_t f = bf16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (uint32_t(vt) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(kPpRows >> 4) << 24);
}
// D += A B with A in tensor memory (16-bit values, two a column).
__device__ __forceinline__ void pp_mma_ta(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, int acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
// A box of 16 rows: of K 64 columns, of V all of them as 64-column halves one behind the other.
__device__ __forceinline__ void pp_tma_k(uint32_t dst, const CUtensorMap *map, int col, int row, int head, int page,
                                         uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(map), "r"(col), "r"(row), "r"(head), "r"(page), "r"(tc_saddr(bar))
      : "memory");
}
// (pp_tma_k also copies Q: a box of tokens x rep heads.)
__device__ __forceinline__ void pp_tma_v(uint32_t dst, const CUtensorMap *map, int row, int head, int page,
                                         uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(map), "r"(0), "r"(row), "r"(0), "r"(head), "r"(page), "r"(tc_saddr(bar))
      : "memory");
}
// 64 or 32 columns of this warp's 32 lanes of tensor memory (a lane a row), waited for.
__device__ __forceinline__ void pp_ld(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
        "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]),
        "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
        "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pp_ld(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
      "}, [%32];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pp_st(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15"
      "};"
      :
      : "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pp_st(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
      "};"
      :
      : "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
// 32 columns of 16 lanes as an MMA's fragment, waited for: r[4 i + e] is column 8 i + 2 (lane % 4) + e % 2 of
// row lane / 4 + 8 (e / 2).
__device__ __forceinline__ void pp_ldo(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15"
      "}, [%16];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pp_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- two floats a register pair
__device__ __forceinline__ uint64_t pp_two(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 pp_split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t pp_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t pp_add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ float pp_max3(float a, float b, float c) {
  float v;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}

__device__ __forceinline__ float pp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a in the low half, b in the high half, rounded to nearest even.
template <bool BF>
__device__ __forceinline__ uint32_t pp_pack(float a, float b) {
  if (BF) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&x);
  }
  const __half2 x = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&x);
}

// Byte offset of V's row r (a multiple of 8) and 64-column half in a stage: boxes one behind the other, in a box
// the halves, in a half its rows of 128 bytes.
template <int HD>
__device__ __forceinline__ int pp_voff(int r, int half, int box) {
  return (r & -box) * (HD * 2) + half * box * 128 + (r & (box - 1)) * 128;
}

// A block of rows and the slots they see: tokens [t0, t1) of a sequence, the token t at slot p0 + t, as
// groups of 16 slots: ga of them from slot 0 on, then those from slot 16 b0 on.
struct PpSpan {
  int row0, t0, t1, p0;          // row0: the q row of token 0
  int lo, first, ga, b0, groups;
  // false: no such block
  __device__ __forceinline__ bool set(const PagedView &c, const PagedQuery &a, const int32_t *starts, int rows,
                                      int max_rows, int i, int tokens, int block, int box) {
    row0 = starts[i];
    const int cnt = starts[i + 1] - row0;
    if (row0 < 0 || row0 > rows || cnt <= 0) return false;
    const int last = min(min(cnt, max_rows), rows - row0);
    if (int64_t(block) * tokens >= last) return false;
    t0 = block * tokens;
    t1 = last - t0 > tokens ? t0 + tokens : last;
    p0 = paged_len(c, i) - cnt;
    const int pmin = p0 + t0, pmax = p0 + t1 - 1;
    lo = a.window > 0 && pmin >= a.window ? pmin - a.window + 1 : 0;
    first = min(a.first, lo);
    // both runs of groups begin at a box's first row (box is a power of two), so no box is cut by a tile's end
    ga = ((first + box - 1) & -box) / kPpGroup;
    b0 = max((lo & -box) / kPpGroup, ga);
    groups = pmax < 0 ? 0 : ga + pmax / kPpGroup + 1 - b0;
    return true;
  }
  __device__ __forceinline__ int slot(int g) const { return (g < ga ? g : g - ga + b0) * kPpGroup; }
  __device__ __forceinline__ int tiles() const { return (groups + kPpGroups - 1) / kPpGroups; }
};

// What a CTA does of one block: tiles [j0, j1) of sequence i, kv head h (-1: the CTA's part is done).
struct PpSeg : PpSpan {
  int i, h, j0, j1;
  int part;  // where unfinished rows go; -1: these are all the block's tiles, the output is written
  __device__ __forceinline__ int halves() const {  // half tiles of 64 slots
    return (min(groups, j1 * kPpGroups) - j0 * kPpGroups + kPpHalfGroups - 1) / kPpHalfGroups;
  }
};

// The block whose first tiles a CTA has and whose last ones it has not: its parts are those of this
// CTA and the `parts` - 1 after it (0: there is none).
struct PpHead {
  int parts, row0, t0, t1, h, pad[3];
};

struct PpArgs {
  PagedView c;
  PagedQuery a;
  const int32_t *starts;
  int rows, max_rows, tokens, blocks, slot_rows;  // tokens: of a tile (128 / rep); blocks: of two tiles, a sequence
  int box;                                        // rows of a TMA box: 16 to 128, at most a page
  PpHead *heads;                                  // [CTAs]
  float2 *part_ml;                                // [2 CTAs][slot_rows]: reference (log2 units) and l
  float *part_o;                                  // [2 CTAs][slot_rows][hd], not divided by l
};

// The line of blocks of one kv head, from sequence 0's first to the last's last; place u is block
// u % blocks of sequence u / blocks, and a place without rows has no length.
__device__ __forceinline__ bool pp_place(const PpArgs &p, int64_t u, PpSpan *sp) {
  return sp->set(p.c, p.a, p.starts, p.rows, p.max_rows, int(u / p.blocks), 2 * p.tokens, int(u % p.blocks), p.box);
}

struct PpShare {
  long long head_len, part, begin, end;  // of one kv head's line, of a CTA's part; this CTA's part
  long long place;                       // where begin falls into the line of its head
  int off;                               // and how many tiles into that block
};

// Measures the line and finds this CTA's part of it (the same on every CTA); all threads.
__device__ __forceinline__ void pp_share(const PpArgs &p, PpShare *sh, long long *sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t n = int64_t(p.c.seqs) * p.blocks, each = (n + kPpThreads - 1) / kPpThreads;
  const int64_t u0 = min(n, tid * each), u1 = min(n, u0 + each);
  long long own = 0;
  PpSpan sp;
  for (int64_t u = u0; u < u1;) {
    if (pp_place(p, u, &sp)) {
      own += sp.tiles() + 1;
      ++u;
    } else {
      u = (u / p.blocks + 1) * p.blocks;  // no further block of this sequence either
    }
  }
  long long upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  long long before = 0, total = 0;
  for (int w = 0; w < kPpThreads / 32; ++w) {
    before += w < warp ? sums[w] : 0;
    total += sums[w];
  }
  const long long line = total * p.c.kv_heads;
  const long long part = max((long long)kPpMinPart, (line + gridDim.x - 1) / gridDim.x);
  const long long begin = min(line, blockIdx.x * part), end = min(line, begin + part);
  if (tid == 0) {
    sh->head_len = total;
    sh->part = part;
    sh->begin = begin;
    sh->end = end;
  }
  if (begin >= end) return;
  long long at = before + upto - own;  // where this thread's places begin
  const long long want = begin % total;
  if (want < at || want >= at + own) return;
  for (int64_t u = u0; u < u1;) {
    if (pp_place(p, u, &sp)) {
      const int len = sp.tiles() + 1;
      if (want < at + len) {
        sh->place = u;
        sh->off = int(want - at);
        return;
      }
      at += len;
      ++u;
    } else {
      u = (u / p.blocks + 1) * p.blocks;
    }
  }
}

template <int HD, bool BF>
__global__ void __launch_bounds__(kPpThreads, PpSmem<HD>::kCtas)
    paged_prompt_kernel(const PpArgs p, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap) {
  using Sm = PpSmem<HD>;
  constexpr int ST = Sm::kStages, NB = Sm::kBufs, CH = Sm::kHeld;
  constexpr int kCopy = kPpSoft / 32, kMma = kCopy + 1, kWalk = kCopy + 3;  // warps
  extern __shared__ __align__(1024) uint8_t pp_sm[];  // the swizzle counts from 1,024-byte lines
  __shared__ uint64_t full[ST], empty[ST], vland, qfull, qempty, segfull[kPpSegs], segempty[kPpSegs];
  __shared__ uint64_t sfull[2][2], pfull[2][2], pvdone[2], ofull[2], ofree[2], done[2];
  __shared__ PpSeg segs[kPpSegs];
  __shared__ PpShare share;
  __shared__ long long sums[kPpThreads / 32];
  __shared__ uint32_t tmem_base;
  __shared__ int dead_flag;
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t *qsm = pp_sm, *ring = pp_sm + 2 * Sm::kTile;
  volatile int *dead = &dead_flag;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      tc_bar_init(&full[s], 1);
      tc_bar_init(&empty[s], 2);  // both tiles' MMAs
    }
    tc_bar_init(&vland, 1);
    tc_bar_init(&qfull, 1);
    tc_bar_init(&qempty, 2);
    for (int s = 0; s < kPpSegs; ++s) {
      tc_bar_init(&segfull[s], 1);
      tc_bar_init(&segempty[s], kPpThreads / 32 - 1);  // every warp but the one that fills them
    }
    for (int x = 0; x < 2; ++x) {
      tc_bar_init(&sfull[x][0], 1);  // a half of the slots each
      tc_bar_init(&sfull[x][1], 1);
      tc_bar_init(&pfull[x][0], 4);
      tc_bar_init(&pfull[x][1], 4);
      tc_bar_init(&pvdone[x], 1);
      tc_bar_init(&ofull[x], 1);
      tc_bar_init(&ofree[x], 4);
    }
    tc_bar_init(&done[0], 1);
    tc_bar_init(&done[1], 1);
    dead_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_saddr(&tmem_base)),
                 "r"(Sm::kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pp_share(p, &share, sums);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  // block k of the CTA's part, once warp 11 has it; seg_done gives its place back
  auto seg_get = [&](int k) -> const PpSeg & {
    pp_wait(&segfull[k % kPpSegs], (k / kPpSegs) & 1, dead, 11);
    return segs[k % kPpSegs];
  };
  auto seg_done = [&](int k) {
    __syncwarp();
    if (lane == 0) tc_arrive(&segempty[k % kPpSegs]);
  };

  if (warp >= kPpSoft / 32) {
    if (Sm::kCtas == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Sm::kRestRegs));
    // One elected thread a warp issues. (Issued by `lane == 0` instead, an MMA took 480 clocks of its warp beside
    // 16 busy ones, against 70: only elect.sync tells the compiler that one thread is left.)
    if (warp == kWalk) {
     if (tc_elect()) {
      // the walk along the CTA's part, and Q
      long long u = share.place, left = share.end - share.begin;
      const long long places = (long long)p.c.seqs * p.blocks;
      int off = share.off, h = share.head_len ? int(share.begin / share.head_len) : 0, nq = 0, k = 0;
      PpHead head{};
      for (;; ++k) {
        PpSeg sg;
        bool some = false;
        while (left > 0 && !some) {
          if (u >= places) {
            u = 0;
            ++h;
          }
          if (!pp_place(p, u, &sg)) {
            u = (u / p.blocks + 1) * p.blocks;
            continue;
          }
          const int nt = sg.tiles();
          const int take = int(min(left, (long long)(nt + 1 - off)));
          sg.i = int(u / p.blocks);
          sg.h = h;
          sg.j0 = min(off, nt);
          sg.j1 = min(off + take, nt);
          sg.part = sg.j0 == 0 && sg.j1 == nt ? -1 : 2 * int(blockIdx.x) + (sg.j0 == 0 ? 1 : 0);
          some = sg.j1 > sg.j0 || nt == 0;
          if (some && sg.j0 == 0 && sg.j1 < nt) {
            const long long first = share.end - left;
            head = PpHead{int((first + nt - 1) / share.part - blockIdx.x + 1), sg.row0, sg.t0, sg.t1, h, {0, 0, 0}};
          }
          left -= take;
          off += take;
          if (off > nt) {
            off = 0;
            ++u;
          }
        }
        if (!some) sg.h = -1;
        if (k >= kPpSegs) pp_wait(&segempty[k % kPpSegs], (k / kPpSegs - 1) & 1, dead, 12);
        if (*dead) break;
        segs[k % kPpSegs] = sg;
        tc_arrive(&segfull[k % kPpSegs]);
        if (!some) break;
        if (sg.j1 > sg.j0) {
          if (nq > 0) pp_wait(&qempty, (nq - 1) & 1, dead, 13);
          if (*dead) break;
          const int two = sg.t1 - sg.t0 > p.tokens ? 2 : 1;
          tc_expect_tx(&qfull, unsigned(two * p.tokens * p.a.rep * HD * 2));
          for (int x = 0; x < two; ++x)
#pragma unroll
            for (int hf = 0; hf < Sm::kHalves; ++hf)
              pp_tma_k(tc_saddr(qsm + x * Sm::kTile + hf * kPpHalf), &qmap, hf * 64, 0, sg.h, sg.row0 + sg.t0 + x * p.tokens,
                       &qfull);
          ++nq;
        }
      }
      if (gridDim.x > 1) p.heads[blockIdx.x] = head;
      // after a wait that ran out: no copy may be in flight when the CTA ends
      if (*dead && nq > 0) tc_wait(&qfull, (nq - 1) & 1, &pp_status_word, 14);
     }
    } else if (warp == kCopy) {
      // K and V of each tile, in turn, a ring stage each. Rows of V that no row of the block sees are zeroed
      // once they are there, by the whole warp; the MMAs hear of the stage after that.
      const bool chosen = tc_elect();
      const int mask = (1 << p.c.shift) - 1;
      const int step = p.box / kPpGroup;          // groups of a box
      int s = 0, turn = 0, lands = 0, fills = 0;  // the next stage, how often the ring has gone round
      for (int k = 0;; ++k) {
        const PpSeg &sg = seg_get(k);
        if (__any_sync(0xffffffffu, *dead || sg.h < 0)) break;
        const int32_t *table = p.c.table + sg.i * p.c.table_stride;
        const int pmax = sg.p0 + sg.t1 - 1;
        int page[kPpGroups];  // of the tile's boxes, read a tile ahead
        auto pages_of = [&](int j) {
#pragma unroll
          for (int u = 0; u < kPpGroups; ++u) {
            const int gg = j * kPpGroups + u * step;
            page[u] = j < sg.j1 && u * step < kPpGroups && gg < sg.groups ? table[sg.slot(gg) >> p.c.shift] : -1;
          }
        };
        auto take = [&]() {  // the next stage, free
          if (turn > 0) pp_wait(&empty[s], (turn - 1) & 1, dead, 15);
          ++fills;
          return s;
        };
        auto next = [&]() {
          if (++s == ST) {
            s = 0;
            ++turn;
          }
        };
        auto copy_k = [&](int j) {
          const int ng = min(kPpGroups, sg.groups - j * kPpGroups), at = take();
          uint8_t *dst = ring + at * Sm::kTile;
          if (chosen && !*dead) {
            tc_expect_tx(&full[at], unsigned((ng + step - 1) / step * p.box * HD * 2));
#pragma unroll
            for (int u = 0; u < kPpGroups; ++u) {
              const int g = u * step;
              if (g >= ng) break;
              const int row = sg.slot(j * kPpGroups + g) & mask;
#pragma unroll
              for (int hf = 0; hf < Sm::kHalves; ++hf)
                pp_tma_k(tc_saddr(dst + hf * kPpHalf + g * (kPpGroup * 128)), &kmap, hf * 64, row, sg.h, page[u], &full[at]);
            }
          }
          next();
        };
        pages_of(sg.j0);
        if (sg.j0 < sg.j1) copy_k(sg.j0);
        for (int j = sg.j0; j < sg.j1; ++j) {
          const int gb = j * kPpGroups, ng = min(kPpGroups, sg.groups - gb);
          const int jb = sg.slot(gb), je = sg.slot(gb + ng - 1) + kPpGroup;
          const bool edge = !(je - 1 <= pmax && (jb >= sg.lo || je <= sg.first));
          const int at = take();
          uint8_t *dst = ring + at * Sm::kTile;
          if (chosen && !*dead) {
            uint64_t *bar = edge ? &vland : &full[at];
            tc_expect_tx(bar, unsigned((ng + step - 1) / step * p.box * HD * 2));
#pragma unroll
            for (int u = 0; u < kPpGroups; ++u) {
              const int g = u * step;
              if (g >= ng) break;
              pp_tma_v(tc_saddr(dst + g * (kPpGroup * HD * 2)), &vmap, sg.slot(gb + g) & mask, sg.h, page[u], bar);
            }
          }
          next();
          pages_of(j + 1);
          if (j + 1 < sg.j1) copy_k(j + 1);
          if (edge) {
            pp_wait(&vland, lands++ & 1, dead, 26);
            for (int g = 0; g < ng; ++g) {
              const int s0 = sg.slot(gb + g);
              if (s0 + kPpGroup - 1 <= pmax && (s0 >= sg.lo || s0 + kPpGroup <= sg.first)) continue;
              for (int e = lane; e < kPpGroup * Sm::kHalves * 8; e += 32) {
                const int r = e / (Sm::kHalves * 8), ch = e % (Sm::kHalves * 8), s1 = s0 + r;
                if (s1 > pmax || (s1 < sg.lo && s1 >= sg.first))
                  *reinterpret_cast<uint4 *>(dst + pp_voff<HD>(g * kPpGroup + r, ch >> 3, p.box) + (ch & 7) * 16) =
                      make_uint4(0, 0, 0, 0);
              }
            }
            tc_fence_proxy();
            __syncwarp();
            if (chosen) tc_arrive(&full[at]);
          }
          if (__any_sync(0xffffffffu, *dead)) break;
        }
        if (__any_sync(0xffffffffu, *dead)) break;
        seg_done(k);
      }
      // after a wait that ran out: no copy may be in flight when the CTA ends
      if (__any_sync(0xffffffffu, *dead)) {
        for (int f = max(0, fills - ST); f < fills; ++f) tc_wait(&full[f % ST], (f / ST) & 1, &pp_status_word, 16);
        if (lands > 0) tc_wait(&vland, (lands - 1) & 1, &pp_status_word, 14);
      }
    } else if (tc_elect()) {
      // The MMAs of tile A (warp kMma) or B (the next): a warp each, since a step's waits and commits take one
      // thread about as long as its MMAs take the tensor cores.
      const int x = warp - kMma;
      const uint32_t ts = tmem + x * 64 * NB, to = tmem + 128 * NB + x * HD;
      // descriptors of the first K-step; the others differ in the address (units of 16 bytes)
      const uint64_t qd = pp_desc(tc_saddr(qsm + x * Sm::kTile), 16);
      const uint64_t kd = pp_desc(tc_saddr(ring), 16), vd = pp_desc(tc_saddr(ring), p.box * 128);
      const uint32_t idv = pp_idesc(BF, HD, true);
      const uint32_t neg = p.a.scale < 0.f ? 1u << 13 : 0u;  // the softmax takes |scale|
      const uint32_t idk = pp_idesc(BF, 0, false) | neg;
      auto scores = [&](int at, int half, int ng) {  // S = +-Q K^T of the ng groups of a half of the stage
        const uint64_t kb = kd + at * (Sm::kTile >> 4) + half * ((kPpHalf / 2) >> 4);
        const uint32_t id = idk | uint32_t(ng * (kPpGroup >> 3)) << 17;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = ((k >> 2) * kPpHalf + (k & 3) * 32) >> 4;
          tc_mma(ts + 64 * (half % NB), qd + off, kb + off, id, k > 0);
        }
      };
      uint32_t vo[kPpGroups];  // V's groups in a stage, in units of 16 bytes
#pragma unroll
      for (int g = 0; g < kPpGroups; ++g) vo[g] = pp_voff<HD>(g * kPpGroup, 0, p.box) >> 4;
      auto values = [&](int at, int half, int ng, int add) {  // O += P V of the ng groups of a half
        const uint64_t vb = vd + at * (Sm::kTile >> 4);
#pragma unroll
        for (int k = 0; k < kPpHalfGroups; ++k)
          if (k < ng) pp_mma_ta(to, ts + 64 * (half % NB) + 8 * k, vb + vo[kPpHalfGroups * half + k], idv, k > 0 ? 1 : add);
      };
      int s = 0, turn = 0;  // the ring, as the copying warp fills it
      auto next = [&]() {
        if (++s == ST) {
          s = 0;
          turn ^= 1;
        }
      };
      int nq = 0, blocks = 0, ph[2] = {0, 0};  // ph: the halves' turns of P
      for (int k = 0;; ++k) {
        const PpSeg &sg = seg_get(k);
        if (*dead || sg.h < 0) break;
        const int n = sg.j1 - sg.j0, nu = sg.halves();
        int left = sg.groups - sg.j0 * kPpGroups;  // groups from this half on
        const bool two = sg.t1 - sg.t0 > p.tokens;
        tc_arrive(&segempty[k % kPpSegs]);
        if (n <= 0) continue;
        ++nq;
        if (x == 1 && !two) {  // tile B has no rows: its part of the stages' release
          for (int v = 0; v < 2 * n; ++v, next()) {
            pp_wait(&full[s], turn, dead, 19);
            tc_arrive(&empty[s]);
          }
          pp_wait(&qfull, (nq - 1) & 1, dead, 17);  // no further ahead of A than a block
          tc_arrive(&qempty);
          continue;
        }
        pp_wait(&qfull, (nq - 1) & 1, dead, 17);
        pp_wait(&full[s], turn, dead, 18);
        tc_fence_after();
        scores(s, 0, min(kPpHalfGroups, left));
        tc_commit(&sfull[x][0]);
        if (NB == 2 && nu > 1) {
          scores(s, 1, min(kPpHalfGroups, left - kPpHalfGroups));
          tc_commit(&sfull[x][1]);
        }
        if (nu <= NB) {
          tc_commit(&empty[s]);
          tc_commit(&qempty);
        } else if (NB == 2) {
          tc_commit(&empty[s]);
        }
        int sk = s;  // the stage of this tile's keys
        next();
        for (int v = 0; v < n; ++v) {
          const int sv = s;
          pp_wait(&full[sv], turn, dead, 19);
          next();  // the next tile's keys
          if (v == 0 && blocks > 0) pp_wait(&ofree[x], (blocks - 1) & 1, dead, 20);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int u = 2 * v + half, buf = half % NB;
            if (u >= nu) break;
            pp_wait(&pfull[x][buf], ph[buf]++ & 1, dead, 21 + half);
            tc_fence_after();
            values(sv, half, min(kPpHalfGroups, left), u > 0);
            left -= kPpHalfGroups;
            // S of half u + NB, which takes this one's place
            const bool here = NB == 1 && half == 0;  // it is of this tile
            const int su = here ? sk : s;
            if (u + NB < nu) {
              if (half == 2 - NB) pp_wait(&full[s], turn, dead, 23);  // its first half
              scores(su, (half + NB) & 1, min(kPpHalfGroups, left - (NB - 1) * kPpHalfGroups));
            }
            // With two halves of S, the last but one turn brings no S and tells only (for a rescale) that P V of this
            // half is done, on a barrier of its own: nothing makes the softmax wait for it, so on sfull the next block's
            // first scores could complete a second phase before a slow softmax warp had looked at the first.
            tc_commit(u + 1 == nu ? &ofull[x] : NB == 2 && u + 2 == nu ? &pvdone[x] : &sfull[x][buf]);
            if (half == 1 || u + 1 == nu) tc_commit(&empty[sv]);
            if (u + NB < nu && (((half + NB) & 1) == 1 || u + NB + 1 == nu)) tc_commit(&empty[su]);
            if (u + NB + 1 == nu) tc_commit(&qempty);
          }
          sk = s;
          if (v + 1 < n) next();
          if (*dead) break;
        }
        ++blocks;
        if (*dead) break;
      }
      tc_commit(&done[x]);
      tc_wait(&done[x], 0, &pp_status_word, 25);
    }
  } else {
    if (Sm::kCtas == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Sm::kSoftRegs));
    const int x = warp >> 2, row = threadIdx.x & 127;
    // row / rep of a row below 128, rep at most 128: 65,536 / rep rounded up is close enough to be exact
    const int rep = p.a.rep, recip = (65536 + rep - 1) / rep;
    auto token_of = [&](int r) { return (r * recip) >> 16; };
    const int rt = token_of(row);  // this thread's token of the tile
    const float scale2 = fmaxf(fabsf(p.a.scale) * kPpLog2e, 1e-37f);
    constexpr float kBias = BF ? 0.f : 7.f;
    const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + x * 64 * NB + lanes, to = tmem + 128 * NB + x * HD + lanes;
    int done_blocks = 0;  // so far
    uint32_t sph = 0;     // bit h: the parity of half h's next S; bit 2: of pvdone's next turn, one a block of two halves or more
    for (int k = 0;; ++k) {
      const PpSeg &sg = seg_get(k);
      if (__any_sync(0xffffffffu, *dead || sg.h < 0)) break;
      const int tok0 = sg.t0 + x * p.tokens, left = min(p.tokens, sg.t1 - tok0);  // the tile's tokens
      if (left <= 0) {  // tile B has no rows
        seg_done(k);
        continue;
      }
      const int pmin = sg.p0 + sg.t0, pmax = sg.p0 + sg.t1 - 1, n = sg.j1 - sg.j0, g0 = sg.j0 * kPpGroups;
      // of this row: its slot (before all of them for a row that is none) and the first slot in the window; of the
      // block's last row the latter, too
      const int pos = rt < left ? sg.p0 + tok0 + rt : -1;
      const bool windowed = p.a.window > 0;
      const int wlo = windowed ? pos - p.a.window + 1 : -(1 << 30);
      const int wmax = windowed ? pmax - p.a.window + 1 : -(1 << 30);
      const int ga = sg.ga, b0 = sg.b0 - sg.ga, groups = sg.groups;
      // groups [whole0, whole1) are seen by every row of the block: slots from wmax to pmin, in one run
      const int whole0 = max(b0 > 0 ? ga : 0, (max(wmax, 0) + kPpGroup - 1) / kPpGroup - b0);
      const int whole1 = (pmin + 1) / kPpGroup - b0;
      float m = -INFINITY, ref = 0.f, l = 0.f;  // m: of the scores as they are; ref: of exp2's argument
      const int nu = sg.halves();
#pragma unroll 1
      for (int u = 0; u < nu; ++u) {
        const int buf = u % NB, gb = g0 + kPpHalfGroups * u;
        const uint32_t tsh = ts + 64 * buf;
        pp_wait(&sfull[x][buf], (sph >> buf) & 1, dead, 24);
        sph ^= 1u << buf;
        tc_fence_after();
        const bool edge = !(gb >= whole0 && gb + kPpHalfGroups <= whole1);  // some rows do not see some slots
        // (Loops stay rolled where registers allow: warps at different places of long straight code wait for
        // instructions. Ragged prompts in a window of 128: 177 us with both loops over parts rolled, 202 unrolled.)
        uint32_t s[CH];
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int part = 0; part < 64; part += CH) {
          pp_ld(tsh + part, s);
          if (edge) {
#pragma unroll
            for (int w = 0; w < CH; w += 32) {
              uint32_t see = 0;  // the visible ones of 32 slots: c <= hi and (c >= lo or c < fi) in each group
#pragma unroll 1
              for (int y = 0; y < 2; ++y) {
                const int gg = gb + (part + w) / kPpGroup + y;
                const int s0 = gg < groups ? kPpGroup * (gg < ga ? gg : gg + b0) : (1 << 30);
                const int hi = min(max(pos - s0 + 1, 0), 16), lo = min(max(wlo - s0, 0), 16);
                const int fi = min(max(p.a.first - s0, 0), 16);
                see |= (((1u << hi) - 1) & (~((1u << lo) - 1) | ((1u << fi) - 1))) << (16 * y);
              }
              if (__all_sync(0xffffffffu, see == 0xffffffffu)) continue;
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!(see & (1u << c))) s[w + c] = 0xff800000u;
            }
            if constexpr (CH < 64) pp_st(tsh + part, s);  // they are read again
          }
#pragma unroll
          for (int c = 0; c < CH; c += 2)
            mx[(c >> 1) & 3] = pp_max3(mx[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
        }
        if (CH < 64 && edge) pp_wait_st();
        const float top = fmaxf(pp_max3(mx[0], mx[1], mx[2]), mx[3]);
        const bool move = (top - m) * scale2 > kPpLazy;
        if (__any_sync(0xffffffffu, move)) {
          float f = 1.f;
          if (move) {
            const float nref = top * scale2 - kBias;
            f = m == -INFINITY ? 0.f : pp_exp2(ref - nref);
            m = top;
            ref = nref;
            l *= f;
          }
          if (u > 0) {
            // O has to be complete up to the last half: this S was issued behind its product, or with two of
            // them the next half's S (behind the last half but one nothing: pvdone)
            if (NB == 2) {
              const bool end = u + 1 == nu;
              pp_wait(end ? &pvdone[x] : &sfull[x][buf ^ 1], (sph >> (end ? 2 : buf ^ 1)) & 1, dead, 30);
              tc_fence_after();
            }
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              float o[16];
              uint32_t w[16];
              tc_ld16(to + c, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * f);
              pp_st(to + c, w);
            }
          }
        }
        uint64_t ls[2] = {0, 0};
        const uint64_t sc2 = pp_two(scale2, scale2), rf2 = pp_two(-ref, -ref);
#pragma unroll 1
        for (int part = 0; part < 64; part += CH) {
          if (CH < 64) pp_ld(tsh + part, s);  // (part's P lies over scores that have been read)
          uint32_t w[CH / 2];
#pragma unroll
          for (int c = 0; c < CH / 2; ++c) {
            const uint64_t x2 = pp_fma2(pp_two(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), sc2, rf2);
            float2 e = pp_split(x2);
            e.x = pp_exp2(e.x);
            e.y = pp_exp2(e.y);
            ls[c & 1] = pp_add2(ls[c & 1], pp_two(e.x, e.y));
            w[c] = pp_pack<BF>(e.x, e.y);
          }
          pp_st(tsh + part / 2, w);
        }
        pp_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) tc_arrive(&pfull[x][buf]);
        const float2 lsum = pp_split(pp_add2(ls[0], ls[1]));
        l += lsum.x + lsum.y;
      }
      if (NB == 2 && nu > 1) sph ^= 4u;
      // The rows: O / l, or what a second kernel makes it of. O is read as an MMA's fragment, 16 rows and 32
      // columns at a time, and a quad's words are transposed, so that rows leave in runs of 64 bytes.
      const int part = sg.part, hq0 = sg.h * rep;
      float f = 1.f;
      if (part < 0) {
        if (p.a.sinks && pos >= 0) l += pp_exp2(p.a.sinks[hq0 + row - rt * rep] * kPpLog2e - ref);
        f = m > -INFINITY ? 1.f / l : 0.f;  // zeros for a row that sees nothing
      } else if (rt < left) {
        p.part_ml[int64_t(part) * p.slot_rows + x * p.tokens * rep + row] = make_float2(m == -INFINITY ? -INFINITY : ref, l);
      }
      if (n > 0) {
        pp_wait(&ofull[x], done_blocks & 1, dead, 27);
        ++done_blocks;
        tc_fence_after();
      }
      const int q = lane & 3;
#pragma unroll 1
      for (int r16 = 0; r16 < 32; r16 += 16) {
        // of the two rows whose pieces this lane handles: where they go, and what they are multiplied by
        uint16_t *out[2];
        float *unfinished[2];
        float fr[2];
        bool there[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int lr = r16 + 8 * b + (lane >> 2), rr = 32 * (warp & 3) + lr;  // the row in the warp, in the tile
          const int tt = token_of(rr);
          fr[b] = __shfl_sync(0xffffffffu, f, lr);
          there[b] = tt < left;
          out[b] = p.a.o + int64_t(sg.row0 + tok0 + tt) * p.a.o_row + (hq0 + rr - tt * rep) * p.a.o_head + 8 * q;
          unfinished[b] = p.part_o + (int64_t(part) * p.slot_rows + x * p.tokens * rep + rr) * HD + 2 * q;
        }
#pragma unroll 1
        for (int col = 0; col < HD; col += 32) {
          uint32_t o[16];
          if (n > 0) {
            pp_ldo(to + (uint32_t(r16) << 16) + col, o);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0u;
          }
          if (part < 0) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              // words of column blocks i; the quad's 4 x 4 words are transposed: lane q gets block q
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = pp_pack<BF>(__uint_as_float(o[4 * i + 2 * b]) * fr[b], __uint_as_float(o[4 * i + 2 * b + 1]) * fr[b]);
#pragma unroll
              for (int i = 0; i < 4; i += 2) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, (q & 1) ? w[i] : w[i + 1], 1);
                if (q & 1) w[i] = got;
                else w[i + 1] = got;
              }
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, (q & 2) ? w[i] : w[i + 2], 2);
                if (q & 2) w[i] = got;
                else w[i + 2] = got;
              }
              if (there[b]) *reinterpret_cast<uint4 *>(out[b] + col) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int b = 0; b < 2; ++b)
              if (there[b])
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  *reinterpret_cast<uint2 *>(unfinished[b] + col + 8 * i) = make_uint2(o[4 * i + 2 * b], o[4 * i + 2 * b + 1]);
          }
        }
      }
      if (n > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) tc_arrive(&ofree[x]);
      }
      seg_done(k);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sm::kTmem) : "memory");
  }
}

constexpr int kPpJoinRows = 16;  // rows a CTA of the joining kernel takes, a warp a row

// Joins the parts of the block that CTA blockIdx.x began and others went on with, in order.
template <int HD, bool BF>
__global__ void __launch_bounds__(128) paged_prompt_join_kernel(const PpArgs p) {
  pdl_trigger();
  pdl_wait();
  const PpHead hd = p.heads[blockIdx.x];
  if (hd.parts <= 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int E = HD / 32;
  for (int r = blockIdx.y * kPpJoinRows + warp; r < (int(blockIdx.y) + 1) * kPpJoinRows; r += 4) {
    const int t = hd.t0 + r / p.a.rep, hq = hd.h * p.a.rep + r % p.a.rep;
    if (t >= hd.t1) return;
    // the first part is what its CTA ended with, the others what theirs began with
    auto at = [&](int s) { return int64_t(2 * (blockIdx.x + s) + (s == 0 ? 1 : 0)) * p.slot_rows + r; };
    const float sink = p.a.sinks ? p.a.sinks[hq] * kPpLog2e : -INFINITY;
    float m = sink;
    for (int s = lane; s < hd.parts; s += 32) m = fmaxf(m, p.part_ml[at(s)].x);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = exp2f(sink - ref), v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int s = 0; s < hd.parts; ++s) {
      const float2 ml = p.part_ml[at(s)];
      const float f = exp2f(ml.x - ref);
      l = fmaf(f, ml.y, l);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = fmaf(f, p.part_o[at(s) * HD + lane * E + e], v[e]);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint16_t *out = p.a.o + int64_t(hd.row0 + t) * p.a.o_row + hq * p.a.o_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t *>(out + e) = pp_pack<BF>(v[e] * inv, v[e + 1] * inv);
  }
}

// ---- host ---------------------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn pp_encoder() {
  static std::atomic<void *> fn{nullptr};
  void *f = fn.load();
  if (!f) {
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      return nullptr;
    fn.store(f);
  }
  return reinterpret_cast<EncodeFn>(f);
}

// The pool as (column, row of a page, head, page), a box of `box` rows x 64 columns (K), or as (column of a
// half, row, half, head, page), a box of `box` rows x all columns, half by half (V); 128-byte swizzle, and
// what lies outside reads as zeros.
bool pp_kv_map(EncodeFn enc, const PagedView &c, bool halves, int box, CUtensorMap *map) {
  const cuuint64_t row = cuuint64_t(c.row_stride) * 2;
  // a dimension of one has no stride of its own
  const cuuint64_t head = c.kv_heads > 1 ? cuuint64_t(c.head_stride) * 2 : row;
  const cuuint64_t page = c.pages > 1 ? cuuint64_t(c.page_stride) * 2 : row;
  const cuuint64_t rows = cuuint64_t(1) << c.shift, heads = cuuint64_t(c.kv_heads), pages = cuuint64_t(c.pages);
  const cuuint64_t kdims[4] = {cuuint64_t(c.hd), rows, heads, pages}, kstr[3] = {row, head, page};
  const cuuint64_t vdims[5] = {64, rows, cuuint64_t(c.hd / 64), heads, pages}, vstr[4] = {row, 128, head, page};
  const cuuint32_t kbox[4] = {64, cuuint32_t(box), 1, 1}, vbox[5] = {64, cuuint32_t(box), cuuint32_t(c.hd / 64), 1, 1};
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  return enc(map, c.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, halves ? 5 : 4,
             halves ? c.v : c.k, halves ? vdims : kdims, halves ? vstr : kstr, halves ? vbox : kbox, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// q as (column, query head of a kv head, kv head, row), a box of 64 columns x rep heads x `tokens` rows.
bool pp_q_map(EncodeFn enc, const PagedView &c, const PagedQuery &a, int rows, int tokens, CUtensorMap *map) {
  const cuuint64_t head = a.heads > 1 ? cuuint64_t(a.q_head) * 2 : 16, row = rows > 1 ? cuuint64_t(a.q_row) * 2 : 16;
  const cuuint64_t dims[4] = {cuuint64_t(c.hd), cuuint64_t(a.rep), cuuint64_t(c.kv_heads), cuuint64_t(rows)};
  const cuuint64_t strides[3] = {head, head * a.rep, row};
  const cuuint32_t box[4] = {64, cuuint32_t(a.rep), 1, cuuint32_t(tokens)}, step[4] = {1, 1, 1, 1};
  return enc(map, c.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<uint16_t *>(a.q), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a call is cut: by sizes alone, so that its scratch can be asked for beforehand.
struct PpPlan {
  int tokens, blocks, ctas, slot_rows, box;
  size_t heads_bytes, ml, po;
};

PpPlan pp_plan(const PagedView &c, int heads, int window, int first, int rows, int max_rows, int max_len, int sms) {
  PpPlan p{};
  const int most = std::min(rows, max_rows), rep = heads / c.kv_heads;
  p.tokens = kPpRows / rep;
  p.blocks = (most + 2 * p.tokens - 1) / (2 * p.tokens);
  p.slot_rows = std::min(2 * p.tokens, most) * rep;
  // The larger a TMA box, the fewer: a box costs about 100 clocks beside its bytes, and 64 KB a tile in boxes of
  // 16 rows (24 of them) took 4,350 clocks, of 32 rows 3,180. But a window's first box begins up to box - 1 slots
  // before it, so short windows take small ones.
  p.box = kPpGroup;
  while (p.box < kPpSlots && 2 * p.box <= (1 << c.shift) && (window == 0 || 16 * p.box <= window)) p.box *= 2;
  // one CTA an SM (two), or fewer when the longest line the sizes allow has fewer parts of kPpMinPart tiles
  int64_t see = max_len;
  if (window > 0) see = std::min<int64_t>(see, int64_t(window) + first + 2 * p.tokens + 2 * p.box);
  const int64_t tiles = (see + kPpSlots - 1) / kPpSlots + 1;
  const int slots = sms * (c.hd == 128 ? PpSmem<128>::kCtas : PpSmem<64>::kCtas);
  const double line = double(p.blocks) * c.kv_heads * c.seqs * double(tiles);
  p.ctas = int(std::max(1.0, std::min(double(slots), line / kPpMinPart + 1.0)));
  if (p.ctas > 1) {
    p.heads_bytes = (size_t(p.ctas) * sizeof(PpHead) + 255) / 256 * 256;
    p.ml = (size_t(2) * p.ctas * p.slot_rows * sizeof(float2) + 255) / 256 * 256;
    p.po = size_t(2) * p.ctas * p.slot_rows * c.hd * sizeof(float);
  }
  return p;
}

struct PpMaps {
  CUtensorMap k, v, q;
};

template <int HD, bool BF>
cudaError_t pp_launch(const PpArgs &p, const PpPlan &plan, const PpMaps &m, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(paged_prompt_kernel<HD, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       PpSmem<HD>::kBytes);
  if (e != cudaSuccess) return e;
  launch_pdl(paged_prompt_kernel<HD, BF>, dim3(plan.ctas), dim3(kPpThreads), PpSmem<HD>::kBytes, st, p, m.k, m.v, m.q);
  if (plan.ctas > 1)
    launch_pdl(paged_prompt_join_kernel<HD, BF>, dim3(plan.ctas, (plan.slot_rows + kPpJoinRows - 1) / kPpJoinRows),
               dim3(128), 0, st, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t paged_status_take(int *code) {
  const int zero = 0;
  *code = 0;
  cudaError_t e = cudaMemcpyFromSymbol(code, pp_status_word, sizeof(int));
  if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(pp_status_word, &zero, sizeof(int));
  if (e == cudaSuccess && !*code && fault_fires(kFaultWait)) *code = 99;  // an injected one
  return e;
}

size_t paged_prompt_scratch(const PagedView &c, int heads, int window, int first, int rows, int max_rows, int max_len,
                            int sms) {
  if (rows < 1 || max_rows < 1) return 0;
  if (paged_few(c, heads, std::min(rows, max_rows))) return paged_few_scratch(c, heads, window, first, rows, max_len, sms);
  const PpPlan p = pp_plan(c, heads, window, first, rows, max_rows, max_len, sms);
  return p.heads_bytes + p.ml + p.po;
}

cudaError_t paged_prompt(const PagedView &c, const PagedQuery &a, const int32_t *starts, int rows, int max_rows,
                         int max_len, void *scratch, int sms, cudaStream_t st) {
  // Few rows leave most of a 128-row tile empty and are bound by the cache's bytes: 5 rows each of 8 sequences
  // over 500 to 2,100 slots (2 query heads a kv head) take 20 us as decode does it, 30 us here.
  if (paged_few(c, a.heads, max_rows)) return paged_few_run(c, a, starts, rows, max_rows, max_len, scratch, sms, st);
  const PpPlan plan = pp_plan(c, a.heads, a.window, a.first, rows, max_rows, max_len, sms);
  EncodeFn enc = pp_encoder();
  if (!enc) return cudaErrorNotSupported;
  PpMaps maps;
  if (!pp_kv_map(enc, c, false, plan.box, &maps.k) || !pp_kv_map(enc, c, true, plan.box, &maps.v) ||
      !pp_q_map(enc, c, a, rows, plan.tokens, &maps.q))
    return cudaErrorInvalidValue;
  uint8_t *base = static_cast<uint8_t *>(scratch);
  const PpArgs p{c, a, starts, rows, max_rows, plan.tokens, plan.blocks, plan.slot_rows, plan.box,
                 reinterpret_cast<PpHead *>(base),
                 reinterpret_cast<float2 *>(base + plan.heads_bytes),
                 reinterpret_cast<float *>(base + plan.heads_bytes + plan.ml)};
  if (c.hd == 128) return c.bf16 ? pp_launch<128, true>(p, plan, maps, st) : pp_launch<128, false>(p, plan, maps, st);
  return c.bf16 ? pp_launch<64, true>(p, plan, maps, st) : pp_launch<64, false>(p, plan, maps, st);
}

}  // namespace hc
