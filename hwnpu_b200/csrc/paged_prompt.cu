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
// (row = token * rep + head). A CTA owns two such tiles (A and B), consecutive tokens of one
// sequence: while the softmax of one runs, the tensor cores work for the other.
//
// Slots come in groups of 16 aligned ones, each inside one page, so a tile of 128 slots is eight TMA
// boxes (a 64-column half for K), from wherever the pages are: first the groups of the first tokens that stay
// visible, then those from the lowest slot any row of the CTA sees to its last token. No tile is
// spent on the slots between. Rows of an edge group that no row of the CTA sees are zeroed in shared
// memory (values only: a hidden score is replaced, but 0 times a hidden NaN would not be 0).
//
//   warps 0-3, 4-7  softmax of tile A, B: a thread owns a row. It reads the row's 128 scores from tensor
//                   memory, keeps the running maximum and sum in float32, writes P back as 16-bit
//                   values over the scores, and at the end O / l to memory
//   warps 8, 10     copy the groups of K, of V (cp.async.bulk.tensor, an mbarrier a ring stage)
//   warp 9          issues the MMAs: S = Q K^T (both operands in shared memory, 128-byte swizzle),
//                   O += P V (P in tensor memory, V in shared memory, MN-major)
//
// Arithmetic. S and O are float32. P = exp2(S scale log2(e) - m) is rounded to the cache's type (the MMA
// wants it of V's type); l sums it unrounded in float32. m is moved only when a score passes it by more
// than 2^8, which rescales O in tensor memory; P is at most 256 then, and fp16's P is held 2^7 higher
// so that its smallest weights stand for 2^-32.
//
// Few rows over a long cache: the tiles of a CTA's rows are split over further CTAs, whose unfinished
// (m, l, O) a second kernel joins, in order.
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
constexpr int kPpThreads = 384;            // three warpgroups: softmax of A, of B, and the rest
// Registers a thread: launched with 168 (65,536 / 384), then 224 for the softmax and 56 for the rest, which
// adds up to the same (2 x 224 + 56 = 3 x 168).
constexpr int kPpSoftRegs = 224, kPpRestRegs = 56;
constexpr int kPpHalf = kPpRows * 128;     // bytes of 128 rows x 64 columns
constexpr float kPpLazy = 8.f;
constexpr float kPpLog2e = 1.4426950408889634f;
constexpr uint32_t kPpTmem = 512;          // columns: S_A, S_B (128 each), O_A, O_B

template <int HD>
struct PpSmem {
  static constexpr int kHalves = HD / 64;
  static constexpr int kTile = kHalves * kPpHalf;  // Q of a tile, or K or V of 128 slots
  // V of a group, [half][16 rows][128 bytes]: a group is one K-step of P V, so its halves may lie together
  static constexpr int kVHalf = kPpGroup * 128;
  static constexpr int kVGroup = kHalves * kVHalf;
  static constexpr int kStages = HD == 128 ? 5 : 10;
  static constexpr int kBytes = (2 + kStages) * kTile + 1024;
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
__device__ __forceinline__ void pp_tma_v(uint32_t dst, const CUtensorMap *map, int row, int head, int page,
                                         uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(map), "r"(0), "r"(row), "r"(0), "r"(head), "r"(page), "r"(tc_saddr(bar))
      : "memory");
}
// 128 columns of this warp's 32 lanes of tensor memory, waited for.
__device__ __forceinline__ void pp_ld128(uint32_t taddr, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,"
      "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
      "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
      "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
      "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127"
      "}, [%128];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
      "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
      "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
      "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
      "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]),
      "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]),
      "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]),
      "=r"(r[63]), "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
      "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]), "=r"(r[80]),
      "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]), "=r"(r[88]), "=r"(r[89]),
      "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]), "=r"(r[96]), "=r"(r[97]), "=r"(r[98]),
      "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]), "=r"(r[104]), "=r"(r[105]), "=r"(r[106]),
      "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]),
      "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]), "=r"(r[120]), "=r"(r[121]), "=r"(r[122]),
      "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(taddr)
      : "memory");
}
// 32 columns, waited for.
__device__ __forceinline__ void pp_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
      "}, [%32];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
      "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
      "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
      "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pp_st32(uint32_t taddr, const uint32_t *r) {
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
__device__ __forceinline__ void pp_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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

// The rows of a CTA and the slots they see: tokens [t0, t1) of sequence i, the token t at slot
// p0 + t, as groups of 16 slots: ga of them from slot 0 on, then those from slot 16 b0 on.
struct PpSpan {
  int row0, t0, t1, p0;          // row0: the q row of token 0
  int lo, first, ga, b0, groups;
  // false: nothing to do
  __device__ __forceinline__ bool set(const PagedView &c, const PagedQuery &a, const int32_t *starts, int rows,
                                      int max_rows, int i, int tokens, int block) {
    row0 = starts[i];
    const int cnt = starts[i + 1] - row0;
    if (row0 < 0 || row0 > rows || cnt <= 0) return false;
    t0 = block * tokens;
    t1 = min(min(t0 + tokens, min(cnt, max_rows)), rows - row0);
    if (t0 >= t1) return false;
    p0 = paged_len(c, i) - cnt;
    const int pmin = p0 + t0, pmax = p0 + t1 - 1;
    lo = a.window > 0 && pmin >= a.window ? pmin - a.window + 1 : 0;
    first = min(a.first, lo);
    ga = (first + kPpGroup - 1) / kPpGroup;
    b0 = max(lo / kPpGroup, ga);
    groups = pmax < 0 ? 0 : ga + pmax / kPpGroup + 1 - b0;
    return true;
  }
  __device__ __forceinline__ int slot(int g) const { return (g < ga ? g : g - ga + b0) * kPpGroup; }
  __device__ __forceinline__ int tiles() const { return (groups + kPpGroups - 1) / kPpGroups; }
  // tiles of one split when the work is cut in up to `splits`
  __device__ __forceinline__ int per(int splits) const { return max(1, (tiles() + splits - 1) / splits); }
};

struct PpArgs {
  PagedView c;
  PagedQuery a;
  const int32_t *starts;
  int rows, max_rows, tokens, blocks, splits;  // tokens: of a tile (128 / rep); blocks: of two tiles
  float *part_ml;                              // [rows][heads][splits][2]: reference (log2 units) and l
  float *part_o;                               // [rows][heads][splits][hd], not divided by l
};

// Copies 128 rows of Q (token-major, heads within) into the swizzled operand; rows past the last token
// are zeros. flip: the sign of a negative scale, which the softmax takes as positive.
template <int HD>
__device__ __forceinline__ void pp_load_q(const PpArgs &p, const PpSpan &sp, int h, int t0, uint8_t *dst, int tid) {
  constexpr int CH = HD / 8;
  const uint32_t flip = p.a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll 4
  for (int u = tid; u < kPpRows * CH; u += kPpRows) {
    const int r = u / CH, ch = u % CH, t = r / p.a.rep, hq = h * p.a.rep + r % p.a.rep;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (t < p.tokens && t0 + t < sp.t1) {
      v = *reinterpret_cast<const uint4 *>(p.a.q + int64_t(sp.row0 + t0 + t) * p.a.q_row + hq * p.a.q_head + 8 * ch);
      v.x ^= flip;
      v.y ^= flip;
      v.z ^= flip;
      v.w ^= flip;
    }
    *reinterpret_cast<uint4 *>(dst + (ch >> 3) * kPpHalf + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
  }
}

template <int HD, bool BF>
__global__ void __launch_bounds__(kPpThreads, 1)
    paged_prompt_kernel(const PpArgs p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using Sm = PpSmem<HD>;
  constexpr int ST = Sm::kStages;
  extern __shared__ uint8_t pp_raw[];
  __shared__ uint64_t full[ST], empty[ST], qfull, sfull[2], pfull[2], ofull[2], done;
  __shared__ uint32_t tmem_base;
  __shared__ int dead_flag;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y, i = blockIdx.z;
  // the last tokens see the most: their CTAs start first
  const int block = p.blocks - 1 - int(blockIdx.x) / p.splits, split = int(blockIdx.x) % p.splits;
  PpSpan sp;
  if (!sp.set(p.c, p.a, p.starts, p.rows, p.max_rows, i, 2 * p.tokens, block)) return;
  const int per = sp.per(p.splits), tiles = sp.tiles();
  const int j0 = split * per, j1 = min(tiles, j0 + per);
  if (j0 >= j1 && split > 0) return;
  const bool alone = tiles <= per;
  const bool two = sp.t1 - sp.t0 > p.tokens;  // tile B has rows
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pp_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *qsm = sm, *ring = sm + 2 * Sm::kTile;
  volatile int *dead = &dead_flag;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      tc_bar_init(&full[s], 1);
      tc_bar_init(&empty[s], 1);
    }
    tc_bar_init(&qfull, two ? 8 : 4);
    for (int x = 0; x < 2; ++x) {
      tc_bar_init(&sfull[x], 1);
      tc_bar_init(&pfull[x], 4);
      tc_bar_init(&ofull[x], 1);
    }
    tc_bar_init(&done, 1);
    dead_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_saddr(&tmem_base)),
                 "r"(kPpTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPpRestRegs));
    if (warp == 8 || warp == 10) {
      // the K (warp 8) or V (warp 10) of each tile, in every other ring stage: for K lane l copies half
      // l % halves of group l / halves, for V lane l both halves of group l
      const bool val = warp == 10;
      const int32_t *table = p.c.table + i * p.c.table_stride;
      const int mask = (1 << p.c.shift) - 1, gi = val ? lane : lane / Sm::kHalves, hf = val ? 0 : lane % Sm::kHalves;
      auto page_of = [&](int j) {
        const int g = j * kPpGroups + gi;
        return j < j1 && gi < kPpGroups && g < sp.groups ? table[sp.slot(g) >> p.c.shift] : -1;
      };
      int page = page_of(j0), fill = val ? 1 : 0;
      for (int j = j0; j < j1; ++j, fill += 2) {
        const int next = page_of(j + 1);
        const int ng = min(kPpGroups, sp.groups - j * kPpGroups);
        const int slot = gi < ng ? sp.slot(j * kPpGroups + gi) : 0;
        const int s = fill % ST;
        if (fill >= ST) pp_wait(&empty[s], (fill / ST - 1) & 1, dead, 11);
        if (*dead) break;
        if (lane == 0) tc_expect_tx(&full[s], unsigned(ng * kPpGroup * HD * 2));
        __syncwarp();
        const uint32_t dst = tc_saddr(ring + s * Sm::kTile);
        if (gi < ng) {
          if (val) pp_tma_v(dst + gi * Sm::kVGroup, &vmap, slot & mask, h, page, &full[s]);
          else pp_tma_k(dst + hf * kPpHalf + gi * (kPpGroup * 128), &kmap, hf * 64, slot & mask, h, page, &full[s]);
        }
        page = next;
      }
      // after a wait that ran out: no copy may be in flight when the CTA ends
      if (*dead)
        for (int f = max(val ? 1 : 0, fill - 2 * ST); f < fill; f += 2)
          tc_wait(&full[f % ST], (f / ST) & 1, &pp_status_word, 12);
    } else if (warp == 9) {
      // descriptors of the first K-step; the others differ in the address (units of 16 bytes)
      const uint64_t qd[2] = {pp_desc(tc_saddr(qsm), 16), pp_desc(tc_saddr(qsm) + Sm::kTile, 16)};
      const uint64_t kd = pp_desc(tc_saddr(ring), 16), vd = pp_desc(tc_saddr(ring), Sm::kVHalf);
      const uint32_t idv = pp_idesc(BF, HD, true);
      auto scores = [&](int x, int s, int ng) {  // S_x = Q_x K^T of the stage's ng groups
        const uint32_t id = pp_idesc(BF, ng * kPpGroup, false);
        const uint64_t kb = kd + s * (Sm::kTile >> 4);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = ((k >> 2) * kPpHalf + (k & 3) * 32) >> 4;
          tc_mma(tmem + x * 128, qd[x] + off, kb + off, id, k > 0);
        }
        tc_commit(&sfull[x]);
      };
      auto values = [&](int x, int s, int ng, bool add) {  // O_x += P_x V
        const uint64_t vb = vd + s * (Sm::kTile >> 4);
#pragma unroll
        for (int k = 0; k < kPpGroups; ++k)
          if (k < ng)
            pp_mma_ta(tmem + 256 + x * 128, tmem + x * 128 + 8 * k, vb + k * (Sm::kVGroup >> 4), idv, add || k > 0);
        tc_commit(&ofull[x]);
      };
      auto groups_of = [&](int j) { return min(kPpGroups, sp.groups - j * kPpGroups); };
      const int n = j1 - j0;
      if (n > 0) {
        pp_wait(&qfull, 0, dead, 13);
        pp_wait(&full[0], 0, dead, 14);
        tc_fence_after();
        if (lane == 0) {
          scores(0, 0, groups_of(j0));
          if (two) scores(1, 0, groups_of(j0));
          tc_commit(&empty[0]);
        }
      }
      const int pmax = sp.p0 + sp.t1 - 1;
      for (int u = 0; u < n; ++u) {
        const int j = j0 + u, ng = groups_of(j), fv = 2 * u + 1, fk = 2 * u + 2;
        pp_wait(&full[fv % ST], (fv / ST) & 1, dead, 15);
        // values of slots that no row of this CTA sees
        const int jb = sp.slot(j * kPpGroups), je = sp.slot(j * kPpGroups + ng - 1) + kPpGroup;
        if (je - 1 > pmax || (jb < sp.lo && je > sp.first)) {
          for (int g = 0; g < ng; ++g) {
            const int s0 = sp.slot(j * kPpGroups + g);
            if (s0 + kPpGroup - 1 <= pmax && (s0 >= sp.lo || s0 + kPpGroup <= sp.first)) continue;
            for (int e = lane; e < kPpGroup * Sm::kHalves * 8; e += 32) {
              const int r = e / (Sm::kHalves * 8), ch = e % (Sm::kHalves * 8), s = s0 + r;
              if (s > pmax || (s < sp.lo && s >= sp.first))
                *reinterpret_cast<uint4 *>(ring + (fv % ST) * Sm::kTile + g * Sm::kVGroup + (ch >> 3) * Sm::kVHalf +
                                           r * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          tc_fence_proxy();
        }
        if (u + 1 < n) pp_wait(&full[fk % ST], (fk / ST) & 1, dead, 16);
        __syncwarp();
        for (int x = 0; x < (two ? 2 : 1); ++x) {
          pp_wait(&pfull[x], u & 1, dead, 17);
          tc_fence_after();
          if (lane == 0) {
            values(x, fv % ST, ng, u > 0);
            if (u + 1 < n) scores(x, fk % ST, groups_of(j + 1));
          }
        }
        if (lane == 0) {
          tc_commit(&empty[fv % ST]);
          if (u + 1 < n) tc_commit(&empty[fk % ST]);
        }
      }
      if (lane == 0) {
        tc_commit(&done);
        tc_wait(&done, 0, &pp_status_word, 18);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPpSoftRegs));
    if (warp < 4 || two) {
      const int x = warp >> 2, row = threadIdx.x & 127;
      pp_load_q<HD>(p, sp, h, sp.t0 + x * p.tokens, qsm + x * Sm::kTile, row);
      tc_fence_proxy();
      __syncwarp();
      if (lane == 0) tc_arrive(&qfull);
      // this thread's row: token t of the sequence, query head hq
      const int rt = row / p.a.rep, t = sp.t0 + x * p.tokens + rt, hq = h * p.a.rep + row % p.a.rep;
      const bool mine = rt < p.tokens && t < sp.t1;
      const int pos = mine ? sp.p0 + t : -1;
      const int wlo = p.a.window > 0 ? pos - p.a.window + 1 : -(1 << 30);  // the first slot in the window
      const float scale2 = fmaxf(fabsf(p.a.scale) * kPpLog2e, 1e-37f);
      constexpr float kBias = BF ? 0.f : 7.f;
      const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
      const uint32_t ts = tmem + x * 128 + lanes, to = tmem + 256 + x * 128 + lanes;
      const int pmin = sp.p0 + sp.t0, pmax = sp.p0 + sp.t1 - 1;
      float m = -INFINITY, ref = 0.f, l = 0.f;  // m: of the scores as they are; ref: of exp2's argument
      for (int u = 0; u < j1 - j0; ++u) {
        const int gb = (j0 + u) * kPpGroups, ng = min(kPpGroups, sp.groups - gb);
        pp_wait(&sfull[x], u & 1, dead, 19);
        tc_fence_after();
        uint32_t s[128];
        pp_ld128(ts, s);
        const int jb = sp.slot(gb), je = sp.slot(gb + ng - 1) + kPpGroup;
        const bool whole = ng == kPpGroups && je - jb == kPpSlots && je - 1 <= pmin &&
                           (p.a.window == 0 || jb > pmax - p.a.window || je <= p.a.first);
        if (!whole) {
#pragma unroll
          for (int g = 0; g < kPpGroups; ++g) {
            const int s0 = g < ng ? sp.slot(gb + g) : (1 << 30);
            const int hi = pos - s0, lo = wlo - s0, fi = p.a.first - s0;  // column c: c <= hi and (c >= lo or c < fi)
#pragma unroll
            for (int c = 0; c < kPpGroup; ++c)
              if (!(c <= hi && (c >= lo || c < fi))) s[g * kPpGroup + c] = 0xff800000u;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kPpSlots; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(s[c]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool move = (top - m) * scale2 > kPpLazy || (m == -INFINITY && top > m);
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
            pp_wait(&ofull[x], (u - 1) & 1, dead, 20);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              pp_ld32(to + c, o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              pp_st32(to + c, o);
            }
          }
        }
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            const float a = pp_exp2(fmaf(__uint_as_float(s[64 * half + c]), scale2, -ref));
            const float b = pp_exp2(fmaf(__uint_as_float(s[64 * half + c + 1]), scale2, -ref));
            ls[c & 2] += a;
            ls[(c & 2) + 1] += b;
            pk[c / 2] = pp_pack<BF>(a, b);
          }
          pp_st32(ts + 32 * half, pk);
        }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        pp_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) tc_arrive(&pfull[x]);
      }
      if (j1 > j0) {
        pp_wait(&ofull[x], (j1 - j0 - 1) & 1, dead, 21);
        tc_fence_after();
      }
      float inv = 1.f;
      const int64_t at = (int64_t(sp.row0 + t) * p.a.heads + hq) * p.splits + split;
      if (alone) {
        if (p.a.sinks && mine) l += pp_exp2(p.a.sinks[hq] * kPpLog2e - ref);
        inv = l > 0.f ? 1.f / l : 0.f;
      } else if (mine) {
        *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(m == -INFINITY ? -INFINITY : ref, l);
      }
      uint16_t *out = p.a.o + int64_t(sp.row0 + t) * p.a.o_row + hq * p.a.o_head;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        if (j1 > j0) {
          pp_ld32(to + c, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (!mine) continue;
        if (alone) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint4 v;
            v.x = pp_pack<BF>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
            v.y = pp_pack<BF>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
            v.z = pp_pack<BF>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
            v.w = pp_pack<BF>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
            *reinterpret_cast<uint4 *>(out + c + e) = v;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4 *>(p.part_o + at * HD + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kPpTmem) : "memory");
  }
}

// Joins the splits of a token's query heads, a warp a head.
template <int HD, bool BF>
__global__ void __launch_bounds__(128) paged_prompt_join_kernel(const PpArgs p) {
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, i = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  PpSpan sp;
  if (!sp.set(p.c, p.a, p.starts, p.rows, p.max_rows, i, 2 * p.tokens, t / (2 * p.tokens)) || t >= sp.t1) return;
  const int per = sp.per(p.splits), used = (sp.tiles() + per - 1) / per;
  if (used <= 1) return;  // the first kernel wrote it
  constexpr int E = HD / 32;
  for (int hq = warp; hq < p.a.heads; hq += 4) {
    const int64_t at = (int64_t(sp.row0 + t) * p.a.heads + hq) * p.splits;
    const float sink = p.a.sinks ? p.a.sinks[hq] * kPpLog2e : -INFINITY;
    float m = sink;
    for (int s = lane; s < used; s += 32) m = fmaxf(m, p.part_ml[2 * (at + s)]);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = lane; s < used; s += 32) l += exp2f(p.part_ml[2 * (at + s)] - ref) * p.part_ml[2 * (at + s) + 1];
    l = warp_sum(l) + exp2f(sink - ref);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int s = 0; s < used; ++s) {
      const float f = exp2f(p.part_ml[2 * (at + s)] - ref);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = fmaf(f, p.part_o[(at + s) * HD + lane * E + e], v[e]);
    }
    uint16_t *out = p.a.o + int64_t(sp.row0 + t) * p.a.o_row + hq * p.a.o_head + lane * E;
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

// The pool as (column, row of a page, head, page), a box of 16 rows x 64 columns (K), or as (column of a
// half, row, half, head, page), a box of 16 rows x all columns, half by half (V); 128-byte swizzle, and
// what lies outside reads as zeros.
bool pp_map(EncodeFn enc, const PagedView &c, bool halves, CUtensorMap *map) {
  const cuuint64_t row = cuuint64_t(c.row_stride) * 2;
  // a dimension of one has no stride of its own
  const cuuint64_t head = c.kv_heads > 1 ? cuuint64_t(c.head_stride) * 2 : row;
  const cuuint64_t page = c.pages > 1 ? cuuint64_t(c.page_stride) * 2 : row;
  const cuuint64_t rows = cuuint64_t(1) << c.shift, heads = cuuint64_t(c.kv_heads), pages = cuuint64_t(c.pages);
  const cuuint64_t kdims[4] = {cuuint64_t(c.hd), rows, heads, pages}, kstr[3] = {row, head, page};
  const cuuint64_t vdims[5] = {64, rows, cuuint64_t(c.hd / 64), heads, pages}, vstr[4] = {row, 128, head, page};
  const cuuint32_t kbox[4] = {64, kPpGroup, 1, 1}, vbox[5] = {64, kPpGroup, cuuint32_t(c.hd / 64), 1, 1};
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  return enc(map, c.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, halves ? 5 : 4,
             halves ? c.v : c.k, halves ? vdims : kdims, halves ? vstr : kstr, halves ? vbox : kbox, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a call is cut: by sizes alone, so that its scratch can be asked for beforehand.
struct PpPlan {
  int tokens, blocks, splits;
  size_t ml, po;  // bytes
};

PpPlan pp_plan(const PagedView &c, int heads, int window, int first, int rows, int max_rows, int max_len, int sms) {
  PpPlan p{};
  if (rows < 1 || max_rows < 1) return p;
  const int most = std::min(rows, max_rows);
  p.tokens = kPpRows / (heads / c.kv_heads);
  p.blocks = (most + 2 * p.tokens - 1) / (2 * p.tokens);
  // The number of splits that ends soonest: waves of CTAs over the SMs times the tiles a CTA walks, with
  // a CTA's start and end counted as kFixed tiles, and the second kernel as as many.
  constexpr int kFixed = 4;
  int64_t see = max_len;
  if (window > 0) see = std::min<int64_t>(see, int64_t(window) + first + std::min(most, 2 * p.tokens));
  const int64_t tiles = std::max<int64_t>(1, (see + kPpSlots - 1) / kPpSlots);
  const int64_t units = int64_t(p.blocks) * c.kv_heads * c.seqs;
  int64_t best = -1;
  p.splits = 1;
  for (int64_t s = 1; s <= std::min<int64_t>(tiles, 64); ++s) {
    const int64_t per = (tiles + s - 1) / s;
    if ((tiles + per - 1) / per != s) continue;
    const int64_t cost = (units * s + sms - 1) / sms * (per + kFixed) + (s > 1 ? kFixed : 0);
    if (best < 0 || cost < best) {
      best = cost;
      p.splits = int(s);
    }
  }
  if (p.splits > 1) {
    p.ml = (size_t(rows) * heads * p.splits * 2 * sizeof(float) + 255) / 256 * 256;
    p.po = size_t(rows) * heads * p.splits * c.hd * sizeof(float);
  }
  return p;
}

template <int HD, bool BF>
cudaError_t pp_launch(const PpArgs &p, const CUtensorMap &km, const CUtensorMap &vm, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(paged_prompt_kernel<HD, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       PpSmem<HD>::kBytes);
  if (e != cudaSuccess) return e;
  launch_pdl(paged_prompt_kernel<HD, BF>, dim3(unsigned(p.blocks) * p.splits, p.c.kv_heads, p.c.seqs), dim3(kPpThreads),
             PpSmem<HD>::kBytes, st, p, km, vm);
  if (p.splits > 1)
    launch_pdl(paged_prompt_join_kernel<HD, BF>, dim3(p.max_rows, p.c.seqs), dim3(128), 0, st, p);
  return cudaGetLastError();
}

}  // namespace

int paged_status_take() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, pp_status_word, sizeof(int)) != cudaSuccess) return 0;
  if (v) cudaMemcpyToSymbol(pp_status_word, &zero, sizeof(int));
  return v;
}

size_t paged_prompt_scratch(const PagedView &c, int heads, int window, int first, int rows, int max_rows, int max_len,
                            int sms) {
  const PpPlan p = pp_plan(c, heads, window, first, rows, max_rows, max_len, sms);
  return p.ml + p.po;
}

cudaError_t paged_prompt(const PagedView &c, const PagedQuery &a, const int32_t *starts, int rows, int max_rows,
                         int max_len, void *scratch, int sms, cudaStream_t st) {
  const PpPlan plan = pp_plan(c, a.heads, a.window, a.first, rows, max_rows, max_len, sms);
  EncodeFn enc = pp_encoder();
  if (!enc) return cudaErrorNotSupported;
  CUtensorMap km, vm;
  if (!pp_map(enc, c, false, &km) || !pp_map(enc, c, true, &vm)) return cudaErrorInvalidValue;
  uint8_t *base = static_cast<uint8_t *>(scratch);
  const PpArgs p{c, a, starts, rows, max_rows, plan.tokens, plan.blocks, plan.splits, reinterpret_cast<float *>(base),
                 reinterpret_cast<float *>(base + plan.ml)};
  if (c.hd == 128) return c.bf16 ? pp_launch<128, true>(p, km, vm, st) : pp_launch<128, false>(p, km, vm, st);
  return c.bf16 ? pp_launch<64, true>(p, km, vm, st) : pp_launch<64, false>(p, km, vm, st);
}

}  // namespace hc
