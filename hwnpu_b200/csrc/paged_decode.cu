// paged_decode.cu: attention of one new token a sequence over a caller's paged 16-bit cache
// (hc_paged_decode_run), and of a few (hc_paged_prompt_run with up to 16 rows of tokens times query heads
// a kv head: a speculative verify): softmax(scale q K^T) V over the visible slots, the cache's
// length split over CTAs and joined (Flash-Decoding, paged.go:227-310).
//
// Bound. A visible slot costs 4 head_dim bytes of HBM (its key and its value, once for all the query
// heads of the kv head) and 4 head_dim flops a query head: at most 8 flops a byte with 8 heads, far
// below the card's balance, so the kernel is bound by HBM and everything else only has to stay out of
// the loads' way.
//
// Split. One CTA a (range of slots, kv head, sequence), 4 warps. The visible slots are taken in groups of 16
// aligned ones (a group never leaves its page: pages have 16 << n slots): first the groups of the
// first tokens that stay visible, then those of the window. A warp takes every fourth group of the
// CTA's range through its own shared-memory ring (cp.async, 16 bytes a lane, no barrier between the
// warps), so that 2 or 3 groups a warp are always in flight. Slots of an edge group that the mask
// hides are filled with zeros instead of being read.
//
// Arithmetic, a group at a time, up to 8 query heads (more take further CTAs, which find the rows in
// the L2 cache):
//   S = Q K^T    mma.sync m16n8k16, rows 0-7 of A the heads, B the key rows by ldmatrix
//   P            exp2(S - m) in float32 with the running maximum m and sum l of each head. m is only
//                moved when a score passes it by more than 2^8 (then O and l are rescaled), which is
//                exact either way: P stays at most 256
//   O += P V     the same MMA: rows 0-7 of A are P rounded to the cache's type, rows 8-15 what the
//                rounding left of P (rounded in its turn), so that the weights carry 16 bits or more
//                at no further MMA; B is V by ldmatrix.trans. O is float32
// Of several tokens both halves of A are rows, and the weights are rounded to the cache's type once.
// The four warps' (m, l, O) are joined in shared memory, the splits' by a second kernel or, up to 8 of them,
// by their cluster over distributed shared memory, all in a fixed order. With `accumulate` the scores are kept in scratch
// (float32, room for the capacity: 4 bytes a slot and query head, so that a sequence past max_len is as fast; scores
// computed over again there took 530 us against 221 for 64 sequences of up to 8,200 and a max_len of 4,000) and
// the visible slots' weights exp2(S - m) / l are summed over the heads once m and l are known.
//
// Measured, on several GPUs. One sequence of 131,071 slots (32 heads over 8 of 128): 90 to 93 us, 5.8 to 6.0 TB/s, 88 to
// 91% of the copy rate. 64 sequences of up to 8,200 with their weights: 203 to 208 us, 5.25 to 5.37 TB/s. 128 in a
// window of 128 (64 heads over 8 of 64): 13 us, 1,024 CTAs of three rounds in two waves; 5 rows each of 8 sequences of
// 500 to 2,100: 18 us, nine rounds and their latencies. With 2 stages and more CTAs an SM: 14.1, 19.8.
#include <cuda_bf16.h>

#include <algorithm>

#include "device.cuh"
#include "kernels.h"
#include "paged.h"

namespace hc {
namespace {

constexpr int kPdWarps = 4;
constexpr int kPdGroup = 16;   // slots of a group
constexpr int kPdHeads = 8;    // query heads a CTA
constexpr int kPdMaxSplits = 256;
constexpr int kPdFew = 16;     // rows of several tokens a CTA
constexpr int kPdCluster = 8;  // splits that a cluster joins
constexpr float kPdLazy = 8.f;  // log2 of how far a score may pass the running maximum
constexpr float kPdLog2e = 1.4426950408889634f;

template <int HD>
struct PdRing {
  static constexpr int kRow = HD * 2;             // bytes of a row
  static constexpr int kHalf = kPdGroup * kRow;   // keys (or values) of a group
  static constexpr int kStage = 2 * kHalf;
  // groups a warp keeps in shared memory, and CTAs an SM
  static constexpr int kStages = 3;
  static constexpr int kCtas = HD == 128 ? 2 : 4;
  static constexpr int kBytes = kPdWarps * kStages * kStage;
  __device__ static __forceinline__ int off(int r, int ch) { return r * kRow + ((ch ^ (r & 7)) << 4); }
};

__device__ __forceinline__ uint32_t pd_saddr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// 16 bytes to shared memory, or 16 zero bytes (nothing is read) when !there.
__device__ __forceinline__ void pd_cp16(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// Two floats at addr of the cluster's CTA `rank`.
__device__ __forceinline__ float2 pd_peer(uint32_t addr, int rank) {
  float2 v;
  asm volatile(
      "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %2, %3;\n ld.shared::cluster.v2.f32 {%0, %1}, [a];\n}\n"
      : "=f"(v.x), "=f"(v.y)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}
__device__ __forceinline__ void pd_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void pd_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void pd_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pd_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <bool TRANS>
__device__ __forceinline__ void pd_ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <bool BF>
__device__ __forceinline__ void pd_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// a in the low half, b in the high half, rounded to nearest even.
template <bool BF>
__device__ __forceinline__ uint32_t pd_pack(float a, float b) {
  if (BF) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&x);
  }
  const __half2 x = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&x);
}
template <bool BF>
__device__ __forceinline__ float2 pd_unpack(uint32_t v) {
  if (BF) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// The sum of P V and of what P's rounding left times V, but P V alone where it is not finite: the rounding may have
// left 0 or less, and an infinite value's product with that would turn the infinity into NaN.
__device__ __forceinline__ float pd_whole(float pv, float left) { return isfinite(pv) ? pv + left : pv; }

// The slots that queries at slots qmin .. n - 1 see, as groups of 16: ga of them from slot 0 on, then those from
// slot 16 b0 on; slot j of them is seen by one of the queries when j < n and (j >= lo or j < first).
struct PdSpan {
  int n, lo, first, ga, b0, groups;
  __device__ __forceinline__ PdSpan(int n_, int qmin, int window, int first_) : n(n_) {
    lo = window > 0 && qmin >= window ? qmin - window + 1 : 0;
    first = min(first_, lo);
    ga = (first + kPdGroup - 1) / kPdGroup;
    b0 = max(lo / kPdGroup, ga);
    groups = n > 0 ? ga + max(0, (n + kPdGroup - 1) / kPdGroup - b0) : 0;
  }
  __device__ __forceinline__ int slot(int g) const { return (g < ga ? g : g - ga + b0) * kPdGroup; }
  __device__ __forceinline__ bool sees(int j) const { return j < n && (j >= lo || j < first); }
  // groups of one split when the work is cut in up to `splits`
  __device__ __forceinline__ int per(int splits) const {
    return max(1, (groups + splits * kPdWarps - 1) / (splits * kPdWarps)) * kPdWarps;
  }
};

struct PdArgs {
  PagedView c;
  PagedQuery a;
  int splits, hgroups;
  bool accumulate, cluster;  // cluster: the splits of a row are one, and join themselves
  int64_t score_stride;  // scores a head keeps in scratch
  float *part_ml;        // [rows][heads][splits][2]: m (log2 units) and l
  float *part_o;         // [rows][heads][splits][hd], not divided by l
  float *scores;         // [seqs][heads][score_stride], log2 units, by group
  const int32_t *starts; // of hc_paged_prompt_run, or null: one row a sequence
  int rows, max_rows;
};

// The rows of sequence i: q rows row0 .. row0 + count - 1, the token t at slot p0 + t.
struct PdRows {
  int row0, count, p0;
  __device__ __forceinline__ PdRows(const PdArgs &p, int i) {
    const int len = paged_len(p.c, i);
    row0 = i;
    count = 1;
    p0 = len - 1;
    if (p.starts) {
      row0 = p.starts[i];
      const int cnt = p.starts[i + 1] - row0;
      const bool there = row0 >= 0 && row0 <= p.rows && cnt > 0;
      count = there ? min(min(cnt, p.max_rows), p.rows - row0) : 0;
      p0 = len - cnt;
    }
  }
  __device__ __forceinline__ PdSpan span(const PdArgs &p) const { return PdSpan(max(0, p0 + count), p0, p.a.window, p.a.first); }
};

// The weights of groups [g0, g1) of (sequence i, kv head h), once each head's m and 1 / l are in ml.
__device__ __forceinline__ void pd_add_weights(const PdArgs &p, const PdSpan &sp, int i, int h, int g0, int g1,
                                               const float2 *ml) {
  float *w = p.c.weights + (int64_t(i) * p.c.kv_heads + h) * p.c.cap;
  const float *s0 = p.scores + (int64_t(i) * p.a.heads + int64_t(h) * p.a.rep) * p.score_stride;
  for (int u = g0 * kPdGroup + threadIdx.x; u < g1 * kPdGroup; u += blockDim.x) {
    const int j = sp.slot(u / kPdGroup) + u % kPdGroup;
    if (!sp.sees(j)) continue;
    float add = 0.f;
    for (int r = 0; r < p.a.rep; ++r) add += exp2f(s0[r * p.score_stride + u] - ml[r].x) * ml[r].y;
    w[j] += add;
  }
}

// MANY: up to 16 rows, the tokens of a sequence times the query heads of a kv head (row = token * rep + head),
// in both halves of A; else the query heads of one token, at most 8.
template <int HD, bool BF, bool MANY>
__global__ void __launch_bounds__(kPdWarps * 32, PdRing<HD>::kCtas) paged_decode_kernel(const PdArgs p) {
  using Ring = PdRing<HD>;
  constexpr int KS = HD / 16;  // k-steps of S = Q K^T
  constexpr int NT = HD / 8;   // column tiles of O
  constexpr int CH = HD / 8;   // 16-byte pieces of a row
  constexpr int RPS = 32 / CH;  // rows a warp copies an instruction
  constexpr int HALVES = MANY ? 2 : 1, ROWS = 8 * HALVES;
  // P is held 2^kBias above exp2(S - m): fp16's smallest weights, 2^-25, then stand for 2^-32, and its
  // largest for 2^15
  constexpr float kBias = BF ? 0.f : 7.f;
  extern __shared__ __align__(128) uint8_t pd_buf[];
  __shared__ float sm_m[kPdWarps][ROWS], sm_l[kPdWarps][ROWS];
  __shared__ float2 sm_ml[ROWS], cl_ml[ROWS];
  __shared__ float sm_f[kPdFew][kPdCluster];
  pdl_trigger();
  pdl_wait();
  const PagedView &c = p.c;
  const int split = blockIdx.x, h = blockIdx.y / p.hgroups, hg = blockIdx.y % p.hgroups, i = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, cq = lane & 3;
  const PdRows rw(p, i);
  if (rw.count <= 0) return;
  const PdSpan sp = rw.span(p);
  const int per = sp.per(p.splits);
  const int g0 = split * per, g1 = min(sp.groups, g0 + per);
  const bool alone = sp.groups <= per;  // one CTA has the whole row
  if (g0 >= g1 && split > 0 && (alone || !p.cluster)) return;
  const int rep = p.a.rep, head0 = h * rep + hg * kPdHeads;
  const int nrows = MANY ? rw.count * rep : min(kPdHeads, rep - hg * kPdHeads);
  // groups that every row sees: below the first one's slot, from the last one's window on
  const int qmin = rw.p0, lo_all = p.a.window > 0 ? rw.p0 + rw.count - p.a.window : 0;

  // the warp's page ids: lane k has that of its k-th group from `at` on, the next 32 are on their way
  const int32_t *table = c.table + i * c.table_stride;
  auto page_of = [&](int k) {
    const int g = g0 + warp + k * kPdWarps;
    return g < g1 ? table[sp.slot(g) >> c.shift] : -1;
  };
  int ids_cur = page_of(lane), ids_nxt = page_of(32 + lane);
  uint8_t *ring = pd_buf + warp * Ring::kStages * Ring::kStage;
  const uint32_t ring_s = pd_saddr(ring);
  const int row0 = lane / CH, ch = lane % CH;
  const int64_t head_off = h * c.head_stride;
  // group k of the warp into its ring; k only grows
  auto issue = [&](int k) {
    const int g = g0 + warp + k * kPdWarps;
    if (k && (k & 31) == 0) {
      ids_cur = ids_nxt;
      ids_nxt = page_of(k + 32 + lane);
    }
    const int page = __shfl_sync(0xffffffffu, ids_cur, k & 31);
    if (g < g1) {
      const int j0 = sp.slot(g);
      const bool in_pool = unsigned(page) < unsigned(c.pages);
      const bool whole = in_pool && j0 + kPdGroup <= sp.n && (j0 >= sp.lo || j0 + kPdGroup <= sp.first);
      const int64_t at = (in_pool ? page : 0) * c.page_stride + head_off +
                         int64_t((j0 & ((1 << c.shift) - 1)) + row0) * c.row_stride + ch * 8;
      const uint16_t *ks = c.k + at, *vs = c.v + at;
      const uint32_t dst = ring_s + (k % Ring::kStages) * Ring::kStage;
#pragma unroll
      for (int s = 0; s < kPdGroup / RPS; ++s) {
        const int r = row0 + s * RPS;
        const bool there = whole || (in_pool && sp.sees(j0 + r));
        pd_cp16(dst + Ring::off(r, ch), ks + s * RPS * c.row_stride, there);
        pd_cp16(dst + Ring::kHalf + Ring::off(r, ch), vs + s * RPS * c.row_stride, there);
      }
    }
    pd_commit();
  };
#pragma unroll
  for (int k = 0; k < Ring::kStages - 1; ++k) issue(k);

  // the rows as A fragments (rows 8-15 are zero for a single token)
  uint32_t qa[KS][2][HALVES];
  int pos[HALVES];  // the rows' slots
#pragma unroll
  for (int b = 0; b < HALVES; ++b) {
    const int r = gq + 8 * b, tok = MANY ? r / rep : 0;
    const bool there = r < nrows;
    const uint16_t *q = p.a.q + int64_t(rw.row0 + tok) * p.a.q_row + (head0 + r - tok * rep) * p.a.q_head + 2 * cq;
    pos[b] = there ? rw.p0 + tok : -1;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qa[s][0][b] = there ? *reinterpret_cast<const uint32_t *>(q + 16 * s) : 0u;
      qa[s][1][b] = there ? *reinterpret_cast<const uint32_t *>(q + 16 * s + 8) : 0u;
    }
  }
  const float scale2 = p.a.scale * kPdLog2e;  // scores in log2 units
  float m[HALVES], l[HALVES];  // of row gq (and gq + 8), the same on its 4 lanes (l: this lane's part)
#pragma unroll
  for (int b = 0; b < HALVES; ++b) {
    m[b] = -INFINITY;
    l[b] = 0.f;
  }
  float o[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
  float *score_row =
      !MANY && p.accumulate && gq < nrows ? p.scores + (int64_t(i) * p.a.heads + head0 + gq) * p.score_stride : nullptr;
  const int lm = lane >> 3, lr = lane & 7;

  for (int k = 0; g0 + warp + k * kPdWarps < g1; ++k) {
    const int g = g0 + warp + k * kPdWarps;
    issue(k + Ring::kStages - 1);
    pd_wait<Ring::kStages - 1>();
    __syncwarp();
    const uint32_t buf = ring_s + (k % Ring::kStages) * Ring::kStage;
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};  // slots 0-7 and 8-15
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      uint32_t b[4];
      pd_ldsm4<false>(buf + Ring::off((lm >> 1) * 8 + lr, 2 * s + (lm & 1)), b);
      const uint32_t q1 = MANY ? qa[s][0][HALVES - 1] : 0u, q3 = MANY ? qa[s][1][HALVES - 1] : 0u;
      pd_mma<BF>(s0, qa[s][0][0], q1, qa[s][1][0], q3, b[0], b[1]);
      pd_mma<BF>(s1, qa[s][0][0], q1, qa[s][1][0], q3, b[2], b[3]);
    }
    const int j0 = sp.slot(g);
    const bool whole = j0 + kPdGroup - 1 <= qmin && (j0 >= lo_all || j0 + kPdGroup <= p.a.first);
    float x[HALVES][4];  // slots 2c, 2c+1, 8+2c, 9+2c
    bool move = false;
    float mx[HALVES];
#pragma unroll
    for (int b = 0; b < HALVES; ++b) {
      x[b][0] = s0[2 * b] * scale2;
      x[b][1] = s0[2 * b + 1] * scale2;
      x[b][2] = s1[2 * b] * scale2;
      x[b][3] = s1[2 * b + 1] * scale2;
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 2 * cq + (e & 1) + 8 * (e >> 1);
          if (!(j <= pos[b] && (p.a.window == 0 || pos[b] - j < p.a.window || j < p.a.first))) x[b][e] = -INFINITY;
        }
      }
      mx[b] = fmaxf(fmaxf(x[b][0], x[b][1]), fmaxf(x[b][2], x[b][3]));
      mx[b] = fmaxf(mx[b], __shfl_xor_sync(0xffffffffu, mx[b], 1));
      mx[b] = fmaxf(mx[b], __shfl_xor_sync(0xffffffffu, mx[b], 2));
      move = move || mx[b] > m[b] + kPdLazy;
    }
    if (score_row) {
      *reinterpret_cast<float2 *>(score_row + g * kPdGroup + 2 * cq) = make_float2(x[0][0], x[0][1]);
      *reinterpret_cast<float2 *>(score_row + g * kPdGroup + 8 + 2 * cq) = make_float2(x[0][2], x[0][3]);
    }
    if (__any_sync(0xffffffffu, move)) {
      float f[2];
#pragma unroll
      for (int b = 0; b < HALVES; ++b) {
        const float nm = fmaxf(m[b], mx[b]);
        f[b] = m[b] == -INFINITY ? 0.f : exp2f(m[b] - nm);
        m[b] = nm;
        l[b] *= f[b];
      }
      if (!MANY) f[1] = f[0];  // what rounding left of rows 0-7 belongs to the same heads
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        o[t][0] *= f[0];
        o[t][1] *= f[0];
        o[t][2] *= f[1];
        o[t][3] *= f[1];
      }
    }
    uint32_t pa[4];
#pragma unroll
    for (int b = 0; b < HALVES; ++b) {
      const float ref = m[b] == -INFINITY ? 0.f : m[b] - kBias;
      float e[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        e[y] = exp2f(x[b][y] - ref);
        l[b] += e[y];
      }
      pa[b] = pd_pack<BF>(e[0], e[1]);
      pa[2 + b] = pd_pack<BF>(e[2], e[3]);
      if (!MANY) {
        const float2 h0 = pd_unpack<BF>(pa[0]), h1 = pd_unpack<BF>(pa[2]);
        pa[1] = pd_pack<BF>(e[0] - h0.x, e[1] - h0.y);
        pa[3] = pd_pack<BF>(e[2] - h1.x, e[3] - h1.y);
      }
    }
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      uint32_t b[4];
      pd_ldsm4<true>(buf + Ring::kHalf + Ring::off((lm & 1) * 8 + lr, t + (lm >> 1)), b);
      pd_mma<BF>(o[t], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
      pd_mma<BF>(o[t + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
    }
    __syncwarp();  // the stage is read before it is filled again
  }
  pd_wait<0>();
  __syncthreads();  // every warp is done with its ring

  // join the warps: [warp][row][hd] float32 in the ring's memory
  float *po = reinterpret_cast<float *>(pd_buf), *cl_o = po + kPdWarps * ROWS * HD;
  static_assert((kPdWarps + 1) * ROWS * HD * sizeof(float) <= Ring::kBytes, "the joined rows lie behind the warps'");
#pragma unroll
  for (int b = 0; b < HALVES; ++b) {
    l[b] += __shfl_xor_sync(0xffffffffu, l[b], 1);
    l[b] += __shfl_xor_sync(0xffffffffu, l[b], 2);
    if (cq == 0) {
      sm_m[warp][gq + 8 * b] = m[b] - kBias;
      sm_l[warp][gq + 8 * b] = l[b];
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float2 v = MANY ? make_float2(o[t][2 * b], o[t][2 * b + 1])
                            : make_float2(pd_whole(o[t][0], o[t][2]), pd_whole(o[t][1], o[t][3]));
      *reinterpret_cast<float2 *>(po + (warp * ROWS + gq + 8 * b) * HD + 8 * t + 2 * cq) = v;
    }
  }
  __syncthreads();
  for (int u = threadIdx.x; u < nrows * (HD / 2); u += kPdWarps * 32) {
    const int r = u / (HD / 2), d = 2 * (u % (HD / 2)), tok = MANY ? r / rep : 0;
    const int hq = head0 + r - tok * rep, row = rw.row0 + tok;
    float mm = sm_m[0][r];
#pragma unroll
    for (int w = 1; w < kPdWarps; ++w) mm = fmaxf(mm, sm_m[w][r]);
    if (alone && p.a.sinks) mm = fmaxf(mm, p.a.sinks[hq] * kPdLog2e);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, vx = 0.f, vy = 0.f;
#pragma unroll
    for (int w = 0; w < kPdWarps; ++w) {
      const float f = exp2f(sm_m[w][r] - ref);
      const float2 v = *reinterpret_cast<const float2 *>(po + (w * ROWS + r) * HD + d);
      ll += f * sm_l[w][r];
      vx += f * v.x;
      vy += f * v.y;
    }
    if (alone) {
      // the heads of one kv head are spread over CTAs: the second kernel adds the weights
      if (p.accumulate && p.hgroups > 1 && d == 0)
        *reinterpret_cast<float2 *>(p.part_ml + 2 * (int64_t(row) * p.a.heads + hq) * p.splits) = make_float2(mm, ll);
      if (p.a.sinks) ll += exp2f(p.a.sinks[hq] * kPdLog2e - ref);
      const float inv = ll > 0.f ? 1.f / ll : 0.f;
      *reinterpret_cast<uint32_t *>(p.a.o + row * p.a.o_row + hq * p.a.o_head + d) = pd_pack<BF>(vx * inv, vy * inv);
      if (d == 0) sm_ml[r] = make_float2(ref, inv);
    } else if (p.cluster) {
      *reinterpret_cast<float2 *>(cl_o + r * HD + d) = make_float2(vx, vy);
      if (d == 0) cl_ml[r] = make_float2(mm, ll);
    } else {
      const int64_t at = (int64_t(row) * p.a.heads + hq) * p.splits + split;
      *reinterpret_cast<float2 *>(p.part_o + at * HD + d) = make_float2(vx, vy);
      if (d == 0) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(mm, ll);
    }
  }
  if (alone) {
    if (!MANY && p.accumulate && p.hgroups == 1) {
      __syncthreads();
      pd_add_weights(p, sp, i, h, 0, sp.groups, sm_ml);
    }
    return;
  }
  if (!p.cluster) return;
  // The cluster's CTAs have the splits of these rows: what each split counts for (8 lanes a row), then a share of the
  // output each, and the weights of the own slots.
  __syncwarp();
  pd_cluster_arrive();
  pd_cluster_wait();
  {
    static_assert(kPdFew * kPdCluster == kPdWarps * 32, "a thread a row and split");
    const int r = threadIdx.x / kPdCluster, s = threadIdx.x % kPdCluster;
    const bool there = r < nrows && s < p.splits;
    const float2 ml = there ? pd_peer(pd_saddr(&cl_ml[min(r, ROWS - 1)]), s) : make_float2(-INFINITY, 0.f);
    const float sink =
        p.a.sinks && r < nrows ? p.a.sinks[head0 + (MANY ? r % rep : r)] * kPdLog2e : -INFINITY;
    float mm = fmaxf(ml.x, sink);
#pragma unroll
    for (int y = 1; y < kPdCluster; y <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, y));
    const float ref = mm == -INFINITY ? 0.f : mm, f = exp2f(ml.x - ref);
    float ll = f * ml.y;
#pragma unroll
    for (int y = 1; y < kPdCluster; y <<= 1) ll += __shfl_xor_sync(0xffffffffu, ll, y);
    ll += exp2f(sink - ref);
    const float inv = ll > 0.f ? 1.f / ll : 0.f;
    sm_f[r][s] = f * inv;
    if (s == 0 && r < nrows) sm_ml[r] = make_float2(ref, inv);
  }
  __syncthreads();
  for (int u = split * (kPdWarps * 32) + threadIdx.x; u < nrows * (HD / 2); u += p.splits * (kPdWarps * 32)) {
    const int r = u / (HD / 2), d = 2 * (u % (HD / 2)), tok = MANY ? r / rep : 0;
    const uint32_t at = pd_saddr(cl_o + r * HD + d);
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int s = 0; s < kPdCluster; ++s) {
      if (s >= p.splits) break;
      const float2 v = pd_peer(at, s);
      x = fmaf(sm_f[r][s], v.x, x);
      y = fmaf(sm_f[r][s], v.y, y);
    }
    *reinterpret_cast<uint32_t *>(p.a.o + (rw.row0 + tok) * p.a.o_row + (head0 + r - tok * rep) * p.a.o_head + d) =
        pd_pack<BF>(x, y);
  }
  __syncwarp();
  pd_cluster_arrive();
  if (!MANY && p.accumulate) pd_add_weights(p, sp, i, h, g0, g1, sm_ml);
  __syncwarp();
  pd_cluster_wait();  // no CTA ends while another reads its rows
}

// m (log2 units) and 1 / l of a query head over all its splits and its sink; by one warp.
__device__ __forceinline__ float2 pd_total(const PdArgs &p, int i, int hq, int used, int lane) {
  const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml) + (int64_t(i) * p.a.heads + hq) * p.splits;
  const float sink = p.a.sinks ? p.a.sinks[hq] * kPdLog2e : -INFINITY;
  float m = sink;
  for (int s = lane; s < used; s += 32) m = fmaxf(m, ml[s].x);
  m = warp_max(m);
  if (m == -INFINITY) return make_float2(0.f, 0.f);
  float l = 0.f;
  for (int s = lane; s < used; s += 32) l += exp2f(ml[s].x - m) * ml[s].y;
  l = warp_sum(l) + exp2f(sink - m);
  return make_float2(m, 1.f / l);
}

// Joins the splits of (sequence, kv head): CTAs x < outs (query heads, times tokens) the output of row x, 4 warps
// taking every fourth split; the others the weights, a share of the groups each.
template <int HD, bool BF>
__global__ void __launch_bounds__(kPdWarps * 32) paged_join_kernel(const PdArgs p, int outs) {
  __shared__ float2 sm_ml[128];
  __shared__ float sm_o[kPdWarps][HD];
  __shared__ float2 sm_f[kPdMaxSplits];
  pdl_trigger();
  pdl_wait();
  const int h = blockIdx.y, i = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rep = p.a.rep;
  const PdRows rw(p, i);
  if (rw.count <= 0) return;
  const PdSpan sp = rw.span(p);
  const int per = sp.per(p.splits), used = max(1, (sp.groups + per - 1) / per);
  const bool alone = used == 1;
  if (int(blockIdx.x) < outs) {
    const int tok = blockIdx.x / rep, hq = h * rep + blockIdx.x % rep, row = rw.row0 + tok;
    if (alone || tok >= rw.count) return;  // the first kernel wrote it
    // every split's m and l in one round of loads, then every split's output in another
    const int64_t at = (int64_t(row) * p.a.heads + hq) * p.splits;
    constexpr int E = HD / 32;
    const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml) + at;
    const float sink = p.a.sinks ? p.a.sinks[hq] * kPdLog2e : -INFINITY;
    for (int s = threadIdx.x; s < used; s += kPdWarps * 32) sm_f[s] = ml[s];
    __syncthreads();
    float m = sink;
    for (int s = lane; s < used; s += 32) m = fmaxf(m, sm_f[s].x);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = lane; s < used; s += 32) l += exp2f(sm_f[s].x - ref) * sm_f[s].y;
    l = warp_sum(l) + exp2f(sink - ref);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 8
    for (int s = warp; s < used; s += kPdWarps) {
      const float f = exp2f(sm_f[s].x - ref);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = fmaf(f, p.part_o[(at + s) * HD + 32 * e + lane], v[e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sm_o[warp][32 * e + lane] = v[e] * inv;
    __syncthreads();
    if (threadIdx.x < HD / 2) {
      const int d = 2 * threadIdx.x;
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kPdWarps; ++w) {
        x += sm_o[w][d];
        y += sm_o[w][d + 1];
      }
      *reinterpret_cast<uint32_t *>(p.a.o + row * p.a.o_row + hq * p.a.o_head + d) = pd_pack<BF>(x, y);
    }
    return;
  }
  if (alone && p.hgroups == 1) return;  // the first kernel added them
  const int wb = gridDim.x - outs, share = (sp.groups + wb - 1) / wb, g0 = (int(blockIdx.x) - outs) * share;
  if (g0 >= sp.groups) return;
  for (int r = warp; r < rep; r += kPdWarps) {
    const float2 tot = pd_total(p, i, h * rep + r, used, lane);
    if (lane == 0) sm_ml[r] = tot;
  }
  __syncthreads();
  pd_add_weights(p, sp, i, h, g0, min(sp.groups, g0 + share), sm_ml);
}

// How a call is cut: by sizes alone, so that its scratch can be asked for beforehand.
struct PdPlan {
  int splits, hgroups, wblocks;
  int64_t score_stride;
  size_t ml, po, scores;  // bytes
  bool cluster, join;     // the splits are joined by their cluster; by a second kernel
};

size_t pd_up(size_t n) { return (n + 255) / 256 * 256; }

// rows: q rows in all; few: of several a sequence (MANY).
PdPlan pd_plan(const PagedView &c, int heads, int window, int first, int rows, bool few, int max_len, bool accumulate,
               int sms) {
  PdPlan p{};
  p.hgroups = few ? 1 : (heads / c.kv_heads + kPdHeads - 1) / kPdHeads;
  auto groups = [&](int len) -> int64_t {
    const int64_t all = (int64_t(len) + kPdGroup - 1) / kPdGroup;
    if (window == 0) return all;
    const int64_t run = int64_t(window) + (few ? kPdFew : 0);
    return std::min<int64_t>(all, (int64_t(first) + kPdGroup - 1) / kPdGroup + (run + kPdGroup - 1) / kPdGroup + 1);
  };
  // The number of splits that ends soonest, in rounds (a group a warp) a CTA walks, its start and its join counted
  // as kFixed rounds, the second kernel as as many. Up to 8 splits that fit at once are clusters, which join their
  // own rows (kJoin rounds): 5 rows each of 8 sequences of 500 to 2,100 slots take 18.2 us so, 19.7 with the
  // second kernel. Clusters that have to wait for room cost more than it (244 us against 206 for 64 sequences of
  // up to 8,200 slots). One sequence: waves of equal CTAs over the SMs. Several, whose lengths the host does not
  // know: where not all CTAs fit at once, all rounds (half of what max_len allows) over the SMs, and then the CTA
  // that ends last, so that a long sequence among short ones is cut (those 64 took 300 us uncut).
  const int64_t units = int64_t(c.seqs) * c.kv_heads * p.hgroups;
  const int64_t slots = int64_t(sms) * (c.hd == 128 ? PdRing<128>::kCtas : PdRing<64>::kCtas);
  constexpr double kFixed = 6, kJoin = 2;
  auto joins = [&](int64_t s) {  // with hgroups a CTA does not have all the heads that give weights
    return s <= kPdCluster && units * s <= slots && (!accumulate || p.hgroups == 1);
  };
  const int64_t rounds = std::max<int64_t>(1, (groups(max_len) + kPdWarps - 1) / kPdWarps);
  double best = -1;
  p.splits = 1;
  for (int64_t s = 1; s <= std::min<int64_t>(rounds, kPdMaxSplits); ++s) {
    const int64_t per = (rounds + s - 1) / s;
    if ((rounds + per - 1) / per != s) continue;
    double cost = s == 1 ? 0 : joins(s) ? kJoin : kFixed;
    if (c.seqs == 1) cost += double((units * s + slots - 1) / slots) * (per + kFixed);
    else cost += (units * s <= slots ? 0 : 0.5 * units * (s * kFixed + rounds) / slots) + per + kFixed;
    if (best < 0 || cost < best) {
      best = cost;
      p.splits = int(s);
    }
  }
  p.score_stride = accumulate ? groups(c.cap) * kPdGroup : 0;
  p.wblocks = accumulate ? int(std::min<int64_t>(64, (groups(max_len) * kPdGroup + 2047) / 2048)) : 0;
  p.cluster = p.splits > 1 && joins(p.splits);
  p.join = (p.splits > 1 && !p.cluster) || (accumulate && p.hgroups > 1);
  if (p.join) {
    p.ml = pd_up(size_t(rows) * heads * p.splits * 2 * sizeof(float));
    p.po = p.splits > 1 ? pd_up(size_t(rows) * heads * p.splits * c.hd * sizeof(float)) : 0;
  }
  p.scores = accumulate ? pd_up(size_t(c.seqs) * heads * p.score_stride * sizeof(float)) : 0;
  return p;
}

template <int HD, bool BF, bool MANY>
cudaError_t pd_launch(const PdArgs &p, const PdPlan &plan, cudaStream_t st) {
  const auto kernel = paged_decode_kernel<HD, BF, MANY>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PdRing<HD>::kBytes);
  if (e != cudaSuccess) return e;
  launch_pdl_cluster(kernel, dim3(plan.splits, p.c.kv_heads * plan.hgroups, p.c.seqs), dim3(kPdWarps * 32),
                     plan.cluster ? plan.splits : 1, PdRing<HD>::kBytes, st, p);
  const int outs = p.a.rep * (MANY ? p.max_rows : 1);
  if (plan.join)
    launch_pdl(paged_join_kernel<HD, BF>, dim3(outs + plan.wblocks, p.c.kv_heads, p.c.seqs), dim3(kPdWarps * 32), 0, st, p,
               outs);
  return cudaGetLastError();
}

template <bool MANY>
cudaError_t pd_run(const PagedView &c, const PagedQuery &a, const int32_t *starts, int rows, int max_rows, int max_len,
                   bool accumulate, void *scratch, int sms, cudaStream_t st) {
  const PdPlan plan = pd_plan(c, a.heads, a.window, a.first, rows, MANY, max_len, accumulate, sms);
  uint8_t *base = static_cast<uint8_t *>(scratch);
  const PdArgs p{c, a, plan.splits, plan.hgroups, accumulate, plan.cluster, plan.score_stride, reinterpret_cast<float *>(base),
                 reinterpret_cast<float *>(base + plan.ml), reinterpret_cast<float *>(base + plan.ml + plan.po), starts,
                 rows, max_rows};
  if (c.hd == 128) return c.bf16 ? pd_launch<128, true, MANY>(p, plan, st) : pd_launch<128, false, MANY>(p, plan, st);
  return c.bf16 ? pd_launch<64, true, MANY>(p, plan, st) : pd_launch<64, false, MANY>(p, plan, st);
}

}  // namespace

size_t paged_decode_scratch(const PagedView &c, int heads, int window, int first, int max_len, bool accumulate, int sms) {
  const PdPlan p = pd_plan(c, heads, window, first, c.seqs, false, max_len, accumulate, sms);
  return p.ml + p.po + p.scores;
}

cudaError_t paged_decode(const PagedView &c, const PagedQuery &a, int max_len, bool accumulate, void *scratch, int sms,
                         cudaStream_t st) {
  return pd_run<false>(c, a, nullptr, c.seqs, 1, max_len, accumulate, scratch, sms, st);
}

bool paged_few(const PagedView &c, int heads, int max_rows) { return int64_t(max_rows) * (heads / c.kv_heads) <= kPdFew; }

size_t paged_few_scratch(const PagedView &c, int heads, int window, int first, int rows, int max_len, int sms) {
  const PdPlan p = pd_plan(c, heads, window, first, rows, true, max_len, false, sms);
  return p.ml + p.po;
}

cudaError_t paged_few_run(const PagedView &c, const PagedQuery &a, const int32_t *starts, int rows, int max_rows,
                          int max_len, void *scratch, int sms, cudaStream_t st) {
  return pd_run<true>(c, a, starts, rows, max_rows, max_len, false, scratch, sms, st);
}

}  // namespace hc
