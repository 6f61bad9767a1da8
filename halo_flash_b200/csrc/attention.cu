// Attention over packed prompts and over a paged K/V cache, one kernel for both, for prompts, chunks and single
// tokens: O = softmax(scale Q K^T + mask) V with grouped heads.
//
// Mathematics. A tile is 128 query rows against KT keys. S = Q K^T goes to TMEM in fp32; each row keeps a
// reference r (near its running maximum) and l = sum of p, p = 2^(c s - c r), c = scale log2 e; O += P V stays in
// TMEM in fp32, and at the end O / l is rounded once. Any reference gives the same result, so r follows the maximum
// only when that has grown by more than 2^8: until then p stays below 2^8 (2^14 in fp16, where all p carry a factor 2^6:
// kLift), which neither type nor the fp32 sums mind, and O need not be rescaled. P is rounded to the inputs' 16-bit type for the tensor cores (as every
// output is), l is summed from the unrounded p.
//
// Rows. The group of query heads that share a K/V head is folded into the rows: row r of a tile is token r / G, head
// r % G, so one token of a group of eight already fills eight rows and K and V are read once for all heads.
//
// Work. A job is one (sequence, K/V head, row tile), costing its number of key tiles plus kJobCost. The jobs in their
// order form one line of cost W, and every CTA takes an equal piece of that line: a job that a border cuts is
// computed in pieces, whose unnormalized sums a second kernel joins. One rule thus balances a prompt's triangle,
// ragged batches, and one long sequence that must be split over the whole GPU. No host knowledge of the lengths is
// needed; every CTA finds its piece from cu / kv_len by itself.
//
// Roles in a CTA (640 threads): warp 16 copies Q, K and V by TMA into shared memory (K and V through a ring of
// stages), one thread of warp 17 issues the tcgen05.mma, warp 18 clears what no row may see of V, and warps 0-15 are two
// pairs of softmax groups. The pairs take alternate key tiles, so that one's exponentials run beside the other's TMEM
// traffic; in a pair thread = row, each group with half of the tile's keys, and the two trade their maxima. (Two groups
// with whole rows of 128 held 208 registers a thread and waited for their own latencies: the exponential unit, 16 a clock,
// was busy 55 % of the time at D = 64.)
//
// Waits are bounded as in stage.cuh: one that runs out sets a flag that makes the other waits return at once, the CTA
// finishes its control flow without storing, and the count is reported by halo_b200_stage_timeouts.
// Barriers without a bound are those that every thread passes equally often whatever the waits said: the one of a pair of
// softmax groups (softmax_pair.cuh) and the CTA's or cluster's at the start and the end. The last one comes after all copies
// and products have landed: also those that were issued behind a wait that had run out.
#include "attention.cuh"

#include <atomic>

#include "common.cuh"
#include "softmax_pair.cuh"
#include "stage.cuh"

namespace halo_b200 {

namespace {

__device__ unsigned int g_attn_timeouts = 0;

constexpr uint32_t kRows = kAttnRows;
constexpr uint32_t kThreads = 640, kSoftmaxWarps = 16;
// Registers: five warpgroups of 96 at launch; the copying and multiplying one gives 32 a thread to the softmax groups,
// which hold half a row of S: 4 x 128 x 104 + 128 x 64 = 640 x 96.
constexpr uint32_t kLaunchRegs = 96, kSoftmaxRegs = 104, kOtherRegs = 64;
static_assert(512 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs, "a share above the launch's total would wait for good");
// What a job costs beside its key tiles, in key tiles. Measured with 1, 2, 3 and 4: 4096 tokens, 16/2 heads of 256: 123, 116, 119,
// 118 us; 8192 tokens, 16/4 heads of 128: 247, 231, 227, 228; of 64: 237, 213, 214, 217; 9 prompts of 5003 tokens: 47.6, 45.4, 44.9,
// 45.2; 24 sessions with 700 new tokens: 84.9, 85.6, 86.5, 87.0.
constexpr uint32_t kJobCost = 2;
constexpr uint32_t kSnap = 1;      // a border within so many tiles of a job's end moves to that end
// Least share of a unit, job costs counted. Measured with 1, 2, 3 and 4: one token over 1501 keys 14.7, 14.2, 14.0, 14.6 us; 4 over
// 513 keys 15.3, 15.2, 15.7, 16.1; 8 over 2049 21.1, 21.0, 21.2, 20.8; 2 over 4097, 32/8 heads of 128: 20.5, 20.6, 20.6, 20.4.
constexpr uint32_t kMinShare = 3;
constexpr uint32_t kMaxCtas = 148;
constexpr float kLazy = 8.0f;      // log2 of the growth that a reference may lag behind
// log2 of a factor on all p, which l has too: in fp16 a p far below the maximum would be subnormal, and 2^(8 + 6) still fits.
template <typename T>
constexpr float kLift = __is_same(T, f16) ? 6.0f : 0.0f;

// CG CTAs (a pair of neighbouring SMs, or one) work on a tile of CG x 128 rows. A pair's tensor cores share the
// operands: each CTA stages half of K (its keys) and half of V (its columns), which halves both the traffic from L2 and
// the reads of shared memory that bound a single CTA at these tile sizes.
template <int D, int CG>
struct Shape {
  static constexpr uint32_t kKeys = D == 256 && CG == 1 ? 64 : 128;    // keys of a tile
  static constexpr uint32_t kStageBytes = kKeys * D * 2 / CG;          // one CTA's share of a tile of K or V
  static constexpr uint32_t kQBytes = kRows * D * 2;
  static constexpr uint32_t kStages = kStageBytes == 32768 ? 4 : 8;
  static constexpr uint32_t kKeyRows = kKeys / CG, kVChunks = D / 64 / CG;
  static constexpr uint32_t kHalf = kKeys / 2;                         // keys of a softmax group, and of a part of P
  // TMEM, 512 columns: buffers of S (which P replaces) from 0, O at the end. With three buffers S(g + 2) is computed while
  // P(g) waits for its product, and neither softmax group waits for S; two leave 128 + 2 x 128 columns at D = 256.
  static constexpr uint32_t kBufs = D <= 128 ? 3 : 2, kAhead = kBufs - 1, kTmemO = 512 - D;
  // Q of the next job is copied ahead where shared memory has room for a second one; where it has not, a job's products
  // are finished before the next one's begin.
  static constexpr uint32_t kQBufs = D <= 128 ? 2 : 1;
  static constexpr bool kDrain = kQBufs == 1;
  static constexpr uint32_t kSlots = kDrain ? 2 : 4;     // references and denominators in flight between the two pairs
};

struct alignas(16) Basics {
  uint32_t tmem, abort;
  unsigned long long drained;  // after a wait has run out: the products issued until then are done
  uint32_t start[4], end[4];  // (sequence, K/V head, row tile, key tile) of the piece's borders
};
template <int D, int CG>
struct alignas(16) Shared : Basics {
  using Sh = Shape<D, CG>;
  unsigned long long kv_full[Sh::kStages], kv_empty[Sh::kStages], q_full[Sh::kQBufs], q_empty[Sh::kQBufs];
  unsigned long long s_full[Sh::kBufs], p_full[Sh::kBufs][2], pv_done[Sh::kBufs], o_empty, v_dirty, v_clean;
  unsigned long long m_full[Sh::kSlots][4], l_full[Sh::kSlots][4];
  float l[Sh::kSlots][kRows];
  float m[Sh::kSlots][kRows];  // references
  PairTrade<kRows> trade[2][kPairTrades];  // what a pair's two groups tell each other
};
template <int D, int CG>
constexpr uint32_t kSmemBytes =
    Shape<D, CG>::kQBufs * Shape<D, CG>::kQBytes + Shape<D, CG>::kStages * Shape<D, CG>::kStageBytes + static_cast<uint32_t>(sizeof(Shared<D, CG>));
static_assert(kSmemBytes<256, 1> <= 232448 && kSmemBytes<256, 2> <= 232448 && kSmemBytes<128, 1> <= 232448 && kSmemBytes<128, 2> <= 232448 &&
                  kSmemBytes<64, 1> <= 232448,
              "shared memory of an SM");

// ---- PTX ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ void bar_init(unsigned long long* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(unsigned long long* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The same barrier in the CTA of rank 0 of the cluster. What it tells of lies in tensor memory, or came by TMA; cluster-scope
// acquire and release on every wait and arrival cost about 300 cycles each (4096 tokens: 234 us instead of 209) and order
// nothing more than that needs. Where a thread's own stores are meant, fence.acq_rel.cluster stands before.
__device__ __forceinline__ void bar_arrive_leader(unsigned long long* b) {
  asm volatile(
      "{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %0, 0;\n"
      "mbarrier.arrive.shared::cluster.b64 _, [r];\n}" ::"r"(smem_addr(b))
      : "memory");
}
// True in one thread of a converged warp. Operands of the tcgen05 instructions live in uniform registers: code that the
// compiler can tell is warp-uniform, with this for a condition, keeps them there.
__device__ __forceinline__ bool elect() {
  uint32_t r;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(kFullMask, v, 0); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// All threads of the CTA, or of both CTAs of a pair.
template <int CG>
__device__ __forceinline__ void sync_all() {
  if constexpr (CG == 2) cluster_sync();
  else __syncthreads();
}
// An arrival on `bar` (in both CTAs of a pair) once the products issued so far are done.
template <int CG>
__device__ __forceinline__ void tc_commit(unsigned long long* bar) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// 32 columns of this warp's 32 TMEM lanes. The results are only valid after tc_wait_ld().
__device__ __forceinline__ void tc_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tc_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tc_wait_ld16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// The waits name the registers of the loads, so that no use of them can move ahead of the wait.
#define HALO_R32(v)                                                                                                       \
  "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),  \
      "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), \
      "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), \
      "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
__device__ __forceinline__ void tc_wait_ld(float (&v)[32]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : HALO_R32(v)::"memory"); }
template <uint32_t N>
__device__ __forceinline__ void tc_wait_ld(float (&v)[N][32]) {
  tc_wait_ld(v[0]);
#pragma unroll
  for (uint32_t i = 1; i < N; ++i) asm volatile("" : HALO_R32(v[i])::"memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
               "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand with 128-byte swizzle (layout type 2, version 1): rows of 128 bytes in groups of eight, 1024
// bytes apart; `lead` is the distance of the next 64 columns, which only an operand contiguous along its M / N axis uses.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) | (static_cast<uint64_t>(1024u >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// fp32 accumulator, A and B both fp16 or both bf16; b_mn: B is contiguous along N.
template <typename T>
__device__ __forceinline__ constexpr uint32_t instr_desc(uint32_t m, uint32_t n, bool b_mn) {
  const uint32_t fmt = sizeof(T) == 2 && __is_same(T, bf16) ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// A bounded wait; a thread whose wait runs out tells the others.
__device__ __forceinline__ void wait(Basics& sh, unsigned long long* b, uint32_t parity) {
  const uint32_t bar = smem_addr(b);
  uint32_t done = 0;
  for (uint32_t spin = 0; spin < kStageSpinLimit && !done; ++spin) {
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (!done && spin >= 64) {
      if (*reinterpret_cast<volatile uint32_t*>(&sh.abort)) return;
      if (spin >= 4096) __nanosleep(256);
    }
  }
  if (!done && atomicExch(&sh.abort, 1u) == 0) atomicAdd(&g_attn_timeouts, 1u);
}
__device__ __forceinline__ bool aborted(Basics& sh) { return *reinterpret_cast<volatile uint32_t*>(&sh.abort) != 0; }

// ---- the line of work -----------------------------------------------------------------------------------------
struct Seq {
  uint32_t row0, rows;  // its query rows
  uint32_t len;         // its keys
  int off;              // row i sees keys [0, off + i + 1) when causal
  uint32_t tiles;       // row tiles
};
__device__ __forceinline__ Seq load_seq(const AttnCall& c, uint32_t b, uint32_t tq) {
  Seq s;
  // lengths that do not fit the buffers are cut, so that no access leaves them
  const uint32_t a0 = min(c.cu[b], c.tokens), a1 = min(c.cu[b + 1], c.tokens);
  s.row0 = a0;
  s.rows = a1 > a0 ? a1 - a0 : 0u;
  s.len = s.rows;
  if (c.kv_len) {
    const unsigned long long room = static_cast<unsigned long long>(c.table_cols) << c.page_shift;
    s.len = static_cast<uint32_t>(min(static_cast<unsigned long long>(c.kv_len[b]), min(room, 0x7FFF0000ull)));
  }
  s.off = static_cast<int>(s.len) - static_cast<int>(s.rows);
  s.tiles = (s.rows + tq - 1) / tq;
  return s;
}
// Keys that row tile i sees.
__device__ __forceinline__ uint32_t key_end(const AttnCall& c, const Seq& s, uint32_t i, uint32_t tq) {
  if (!c.causal) return s.len;
  const int e = s.off + static_cast<int>(min(s.rows, (i + 1) * tq));
  return e > 0 ? static_cast<uint32_t>(e) : 0u;
}
// sum over i < n of floor((a i + b) / M) for a power of two M. a n + b < 2^32. The well-known count of the lattice points
// under a line: the parts that divide are taken out, the axes trade places, as in Euclid's algorithm on (a, M).
template <uint32_t M>
__device__ __forceinline__ unsigned long long floor_sum(uint32_t n, uint32_t a, uint32_t b) {
  auto pairs = [](uint32_t k) { return static_cast<unsigned long long>(k) * (k - 1) / 2; };
  unsigned long long s = pairs(n) * (a / M) + static_cast<unsigned long long>(n) * (b / M);
  a %= M;
  uint32_t y = a * n + b % M, m = M;
  while (y >= m) {  // the sum's lattice points seen along the other axis; a < m here
    n = y / m;
    const uint32_t rest = y - n * m, q = m / a, r = rest / a;
    s += pairs(n) * q + static_cast<unsigned long long>(n) * r;
    const uint32_t next = m - q * a;
    m = a;
    a = next;
    y = a * n + (rest - r * m);
  }
  return s;
}
// Cost of the first x row tiles of a sequence (one K/V head).
template <uint32_t KT>
__device__ __forceinline__ unsigned long long cost_before(const AttnCall& c, const Seq& s, uint32_t x, uint32_t tq) {
  unsigned long long w = static_cast<unsigned long long>(x) * kJobCost;
  if (x == 0) return w;
  if (!c.causal) return w + static_cast<unsigned long long>(x) * ((s.len + KT - 1) / KT);
  if (x == s.tiles) w += (s.len + KT - 1) / KT, --x;  // the last tile may be short
  // the others end at off + (i + 1) tq, those up to i0 at or before key 0
  uint32_t i0 = 0;
  if (s.off < 0) i0 = static_cast<uint32_t>(-s.off) / tq;
  if (x > i0)
    w += floor_sum<KT>(x - i0, tq, static_cast<uint32_t>(s.off + static_cast<int>((i0 + 1) * tq) + static_cast<int>(KT) - 1));
  return w;
}

// One warp: where the line of work is cut for unit x of `units` (as many as there is work for), as (sequence, head, row
// tile, key tile); (batch, 0, 0, 0) behind the last job. A border inside a job's fixed cost or near its end moves to the
// job's own border.
template <uint32_t KT>
__device__ void find_border(const AttnCall& c, uint32_t x, uint32_t units, uint32_t tq, uint32_t (&at)[4]) {
  const uint32_t lane = threadIdx.x & 31u;
  Seq s = {};
  unsigned long long w = 0, all = 0, sum = 0;
  auto weigh = [&](uint32_t b0) {  // this lane's sequence, and the running sum over the warp
    w = 0;
    if (b0 + lane < c.batch) {
      s = load_seq(c, b0 + lane, tq);
      w = cost_before<KT>(c, s, s.tiles, tq) * c.kv_heads;
    }
    sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long t = __shfl_up_sync(kFullMask, sum, o);
      if (lane >= static_cast<unsigned>(o)) sum += t;
    }
    return __shfl_sync(kFullMask, sum, 31);
  };
  // the last group is weighed first and the first one last, where it is needed next
  for (uint32_t b0 = (c.batch - 1) / 32 * 32;; b0 -= 32) {
    all += weigh(b0);
    if (b0 == 0) break;
  }
  at[0] = c.batch, at[1] = at[2] = at[3] = 0;
  const unsigned long long most = (all + kMinShare - 1) / kMinShare;
  const uint32_t n = most < units ? static_cast<uint32_t>(most) : units;
  if (x >= n) return;
  unsigned long long u = all / n * x + all % n * x / n;
  for (uint32_t b0 = 0; b0 < c.batch; b0 += 32) {
    const unsigned long long here = b0 ? weigh(b0) : __shfl_sync(kFullMask, sum, 31);
    if (u >= here) {
      u -= here;
      continue;
    }
    const int src = __ffs(__ballot_sync(kFullMask, sum > u)) - 1;
    const uint32_t bb = b0 + static_cast<uint32_t>(src);
    const unsigned long long per_head = __shfl_sync(kFullMask, w, src) / c.kv_heads;
    unsigned long long rest = u - __shfl_sync(kFullMask, sum - w, src);
    s.row0 = __shfl_sync(kFullMask, s.row0, src);
    s.rows = __shfl_sync(kFullMask, s.rows, src);
    s.len = __shfl_sync(kFullMask, s.len, src);
    s.off = __shfl_sync(kFullMask, s.off, src);
    s.tiles = __shfl_sync(kFullMask, s.tiles, src);
    uint32_t h = 0;
    while (h + 1 < c.kv_heads && rest >= per_head) rest -= per_head, ++h;
    uint32_t lo = 0, hi = s.tiles;  // cost_before(lo) <= rest < cost_before(hi)
    unsigned long long before = 0;
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo + 31) / 32, mid = lo + step * (lane + 1);
      const unsigned long long cost = mid < hi ? cost_before<KT>(c, s, mid, tq) : ~0ull;
      const int f = __ffs(__ballot_sync(kFullMask, cost > rest)) - 1;  // the last lane's always is
      if (f > 0) before = __shfl_sync(kFullMask, cost, f - 1);
      lo += step * static_cast<uint32_t>(f);
      hi = min(hi, lo + step);
    }
    uint32_t i = lo;
    rest -= before;
    const uint32_t n_keys = (key_end(c, s, i, tq) + KT - 1) / KT;
    uint32_t t = rest <= kJobCost ? 0u : static_cast<uint32_t>(rest) - kJobCost;
    if (t > 0 && t + kSnap >= n_keys) {
      t = 0;
      if (++i == s.tiles) {
        i = 0;
        if (++h == c.kv_heads) {
          h = 0;
          // the next sequence that has rows
          uint32_t nb = bb + 1;
          while (nb < c.batch && load_seq(c, nb, tq).rows == 0) ++nb;
          at[0] = nb;
          return;
        }
      }
    }
    at[0] = bb, at[1] = h, at[2] = i, at[3] = t;
    return;
  }
}

// The pieces of jobs between two borders, one after the other.
template <uint32_t KT>
struct Pieces {
  const AttnCall& c;
  uint32_t tq, b, h, i, t;
  uint32_t eb, eh, ei, et;
  Seq s;
  // the present piece
  uint32_t t0, t1, n, keys;
  __device__ __forceinline__ Pieces(const AttnCall& call, const Basics& sh, uint32_t tq_) : c(call), tq(tq_) {
    b = sh.start[0], h = sh.start[1], i = sh.start[2], t = sh.start[3];
    eb = sh.end[0], eh = sh.end[1], ei = sh.end[2], et = sh.end[3];
    if (b < c.batch) s = load_seq(c, b, tq);
  }
  __device__ __forceinline__ bool next() {
    while (true) {
      if (b >= c.batch) return false;
      if (s.rows == 0) {  // nothing to do for this sequence
        if (b == eb) return false;
        ++b;
        h = i = t = 0;
        if (b < c.batch) s = load_seq(c, b, tq);
        continue;
      }
      break;
    }
    const bool last = b == eb && h == eh && i == ei;
    if (last && t >= et) return false;
    keys = key_end(c, s, i, tq);
    n = (keys + KT - 1) / KT;
    t0 = t;
    t1 = last ? min(et, n) : n;
    return true;
  }
  // Behind the present piece.
  __device__ __forceinline__ void advance() {
    if (b == eb && h == eh && i == ei) {
      t = et;
      return;
    }
    t = 0;
    if (++i == s.tiles) {
      i = 0;
      if (++h == c.kv_heads) {
        h = 0;
        ++b;
        if (b < c.batch) s = load_seq(c, b, tq);
      }
    }
  }
};

// ---- the kernel -------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<bf16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<f16>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <uint32_t V>
struct Int {
  static constexpr uint32_t value = V;
};

// The 4 x 4 exchange among four neighbouring lanes: u[j] becomes part (lane & 3) of lane (lane & ~3) + j.
__device__ __forceinline__ void trade4(uint4 (&u)[4], uint32_t lane) {
#pragma unroll
  for (uint32_t bit = 1; bit <= 2; bit <<= 1) {
    const bool up = (lane & bit) != 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      if (i & bit) continue;
      uint4 t = up ? u[i] : u[i + bit];
      t.x = __shfl_xor_sync(kFullMask, t.x, bit);
      t.y = __shfl_xor_sync(kFullMask, t.y, bit);
      t.z = __shfl_xor_sync(kFullMask, t.z, bit);
      t.w = __shfl_xor_sync(kFullMask, t.w, bit);
      if (up) u[i] = t;
      else u[i + bit] = t;
    }
  }
}

template <typename T, int D, int CG>
__global__ void __launch_bounds__(kThreads, 1)
    attention_kernel(const __grid_constant__ AttnCall c, const __grid_constant__ CUtensorMap qmap,
                     const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using Sh = Shape<D, CG>;
  constexpr uint32_t KT = Sh::kKeys, ST = Sh::kStages, kChunks = D / 64, NB = Sh::kBufs, NQ = Sh::kQBufs, NS = Sh::kSlots;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  auto& sh = *reinterpret_cast<Shared<D, CG>*>(smem_raw + NQ * Sh::kQBytes + ST * Sh::kStageBytes);
  const uint32_t q_smem = smem_addr(smem_raw), kv_smem = q_smem + NQ * Sh::kQBytes;
  const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31u;
  const uint32_t rank = CG == 2 ? blockIdx.x & 1u : 0u, unit = blockIdx.x / CG, units = gridDim.x / CG;
  const uint32_t tq_cta = kRows / c.group, tq = CG * tq_cta;  // tokens of a CTA's rows, of a row tile

  if (threadIdx.x == 0) {
    // a pair's products need both CTAs' operands: the leader's barriers count the other's arrivals too
    const uint32_t both = rank == 0 ? CG : 1;
    for (uint32_t i = 0; i < ST; ++i) bar_init(&sh.kv_full[i], both), bar_init(&sh.kv_empty[i], 1);
    for (uint32_t i = 0; i < NQ; ++i) bar_init(&sh.q_full[i], both), bar_init(&sh.q_empty[i], 1);
    bar_init(&sh.v_dirty, 1);
    bar_init(&sh.v_clean, 1);
    bar_init(&sh.o_empty, 8 * CG);
    for (uint32_t i = 0; i < NB; ++i) {
      bar_init(&sh.s_full[i], 1);
      for (uint32_t w = 0; w < 2; ++w) bar_init(&sh.p_full[i][w], 4 * CG);
      bar_init(&sh.pv_done[i], 1);
    }
    for (uint32_t i = 0; i < NS; ++i)
      for (int w = 0; w < 4; ++w) bar_init(&sh.m_full[i][w], 1), bar_init(&sh.l_full[i][w], 1);
    bar_init(&sh.drained, 1);
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kSoftmaxWarps + 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sh.tmem)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sh.tmem)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  if (threadIdx.x < 3) {
    const CUtensorMap* map = threadIdx.x == 0 ? &qmap : threadIdx.x == 1 ? &kmap : &vmap;
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  pdl_wait_and_trigger();
  if (warp < 2) {
    // this unit's borders: warp 0 finds the first, warp 1 the last
    uint32_t at[4];
    find_border<KT>(c, unit + warp, units, tq, at);
    if (lane < 4) (warp ? sh.end : sh.start)[lane] = lane == 0 ? at[0] : lane == 1 ? at[1] : lane == 2 ? at[2] : at[3];
  }
  tc_before();
  sync_all<CG>();
  tc_after();
  const uint32_t tmem = sh.tmem;

  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    Pieces<KT> pc(c, sh, tq);
    if (warp == kSoftmaxWarps) {
      // ---- copies -------------------------------------------------------------------------------------------------
      uint32_t job = 0;
      uint32_t issued = 0;  // stages that have had a load
      const uint32_t q_bytes = tq_cta * c.group * 128u * kChunks;
      uint32_t st = 0, ph = 1;  // the next stage, and the parity of its kv_empty phase (a new barrier's phase before the first is over)
      const uint32_t shift = c.box_shift, page_mask = (1u << c.page_shift) - 1u, vcol = uniform(rank * (D / CG));
      // One operand's tile: up to `kMost` key rows from key0 (of the sequence) on, kCh chunks of 64 columns from `col` on,
      // laid out [chunk][row], in boxes of rows that lie in one page; lane first + x holds the page of box x. An elected
      // thread issues the copies.
      auto load_kv = [&](auto most, auto chunks, const CUtensorMap* map, uint32_t row0, uint32_t h, uint32_t key0, uint32_t keys, uint32_t col,
                         uint32_t pages, uint32_t first) {
        constexpr uint32_t kMost = decltype(most)::value, kCh = decltype(chunks)::value;
        // rows behind the last visible key are left out by whole boxes
        const uint32_t rows = keys > key0 ? min(kMost, keys - key0) : 0u, boxes = uniform((rows + (1u << shift) - 1u) >> shift);
        const uint32_t us = uniform(st), bar = smem_addr(&sh.kv_full[0]) + us * 8u, base = kv_smem + us * Sh::kStageBytes, hh = uniform(h);
        const uint32_t row = uniform(c.table ? key0 & page_mask : row0 + key0);
        const uint32_t page0 = __shfl_sync(kFullMask, pages, first), page1 = __shfl_sync(kFullMask, pages, first + 1);
        wait(sh, &sh.kv_empty[st], ph);
        if (aborted(sh)) return;
        issued |= 1u << st;
        auto box = [&](uint32_t x, uint32_t r, uint32_t page) {
#pragma unroll
          for (uint32_t ch = 0; ch < kCh; ++ch)
            tma_4d(base + (ch * kMost + (x << shift)) * 128u, map, static_cast<int>(col + ch * 64), static_cast<int>(r), static_cast<int>(hh),
                   static_cast<int>(page), bar);
        };
        if (elect()) {
          stage_expect(bar, (boxes << shift) * 128u * kCh);
          if (boxes > 0) box(0, row, page0);
          if (boxes > 1) box(1, c.table ? (row + (1u << shift)) & page_mask : row + (1u << shift), page1);
        }
        __syncwarp();
        for (uint32_t x = 2; x < boxes; ++x) {  // pages of less than 64 rows
          const uint32_t page = __shfl_sync(kFullMask, pages, first + x), r = c.table ? (row + (x << shift)) & page_mask : row + (x << shift);
          if (elect()) box(x, r, page);
          __syncwarp();
        }
        if (++st == ST) st = 0, ph ^= 1u;
      };
      // Each lane looks up the page of one box of a tile, a tile ahead of its use.
      auto look_up = [&](uint32_t t) -> uint32_t {
        const uint32_t key = t * KT + (lane << shift);
        return c.table && key < min(pc.keys, (t + 1) * KT) ? static_cast<uint32_t>(c.table[pc.b * c.table_stride + (key >> c.page_shift)]) : 0u;
      };
      // The order of use, which is also the order of the stages: K(g), V(g - kAhead), ..., what is left of V at the end
      // (and, where Q has one buffer, at the end of each job).
      struct Tile {
        uint32_t row0, h, t, keys, pages;
      } last[Sh::kAhead];
      uint32_t left = 0;  // tiles whose V is still to come
      auto load_v = [&] {
        const Tile& v = left == 1 ? last[0] : last[Sh::kAhead - 1];
        load_kv(Int<KT>{}, Int<Sh::kVChunks>{}, &vmap, v.row0, v.h, v.t * KT, v.keys, vcol, v.pages, 0);
        --left;
      };
      for (; pc.next() && !aborted(sh); pc.advance()) {
        uint32_t ahead = pc.t0 < pc.t1 ? look_up(pc.t0) : 0u;
        for (uint32_t t = pc.t0; t < pc.t1; ++t) {
          const uint32_t pages = ahead;
          if (t + 1 < pc.t1) ahead = look_up(t + 1);
          if (t == pc.t0) {
            if constexpr (Sh::kDrain)
              while (left) load_v();
            const uint32_t qb = uniform(job % NQ);
            if (job >= NQ) wait(sh, &sh.q_empty[qb], (job / NQ - 1) & 1u);
            if (aborted(sh)) break;
            const uint32_t bar = uniform(smem_addr(&sh.q_full[qb])), head = uniform(pc.h * c.group), tok = uniform(pc.s.row0 + pc.i * tq + rank * tq_cta);
            const uint32_t to = uniform(q_smem + qb * Sh::kQBytes);
            if (elect()) {
              stage_expect(bar, q_bytes);
#pragma unroll
              for (uint32_t ch = 0; ch < kChunks; ++ch)
                tma_3d(to + ch * kRows * 128u, &qmap, static_cast<int>(ch * 64), static_cast<int>(head), static_cast<int>(tok), bar);
            }
            __syncwarp();
            ++job;
          }
          load_kv(Int<Sh::kKeyRows>{}, Int<kChunks>{}, &kmap, pc.s.row0, pc.h, t * KT + rank * Sh::kKeyRows, pc.keys, 0, pages,
                  rank * (Sh::kKeyRows >> shift));
          if (left == Sh::kAhead) load_v();
#pragma unroll
          for (uint32_t i = Sh::kAhead - 1; i > 0; --i) last[i] = last[i - 1];
          last[0] = Tile{pc.s.row0, pc.h, t, pc.keys, pages};
          ++left;
        }
      }
      while (left && !aborted(sh)) load_v();
      // every stage's last use is over before the CTA may leave: no arrival of the other CTA's products is under way
      if (!aborted(sh)) {
        for (uint32_t i = 0; i < ST; ++i) {
          wait(sh, &sh.kv_empty[st], ph);
          if (++st == ST) st = 0, ph ^= 1u;
        }
        for (uint32_t i = job > NQ ? job - NQ : 0u; i < job; ++i) wait(sh, &sh.q_empty[i % NQ], (i / NQ) & 1u);
      }
      if (aborted(sh)) {
        // no copy may land in shared memory that another CTA owns by then: one more bounded wait for each
        for (uint32_t st = 0; st < ST; ++st)
          if (issued >> st & 1u) {
            stage_wait(smem_addr(&sh.kv_full[st]), 0);
            stage_wait(smem_addr(&sh.kv_full[st]), 1);
          }
        for (uint32_t i = 0; i < min(job, NQ); ++i) {
          stage_wait(smem_addr(&sh.q_full[i]), 0);
          stage_wait(smem_addr(&sh.q_full[i]), 1);
        }
      }
    } else if (warp == kSoftmaxWarps + 1 && rank == 0) {
      // ---- matrix products, issued by one thread (of the pair) -----------------------------------------------------
      constexpr uint32_t idesc_s = instr_desc<T>(CG * kRows, KT, false), idesc_o = instr_desc<T>(CG * kRows, D, true);
      const uint32_t qs = uniform(q_smem), kvs = uniform(kv_smem), tm = uniform(tmem);
      uint32_t g = 0, job = 0, tails = 0, st = 0, ph = 0;  // the stages are used in the order in which they are filled
      uint32_t sb = 0, pb = 0, pph = 0;                    // buffer of the next S, of the next P, and its phase
      uint32_t left = 0;                                   // tiles whose P V is still to come
      struct Tile {
        uint32_t first, tail, job;
      } last[Sh::kAhead];
      auto next_stage = [&] {
        if (++st == ST) st = 0, ph ^= 1u;
      };
      auto pv = [&] {
        const Tile& v = left == 1 ? last[0] : last[Sh::kAhead - 1];
        const uint32_t buf = uniform(pb), acc = uniform(v.first) ^ 1u;
        const uint64_t d = smem_desc(kvs + uniform(st) * Sh::kStageBytes, KT * 128u);
        wait(sh, &sh.kv_full[st], ph);
        if (v.tail) {
          if (lane == 0) bar_arrive(&sh.v_dirty);
          wait(sh, &sh.v_clean, tails++ & 1u);
        }
        if (v.first && v.job > 0) wait(sh, &sh.o_empty, (v.job - 1) & 1u);
#pragma unroll
        for (uint32_t part = 0; part < 2; ++part) {
          wait(sh, &sh.p_full[buf][part], pph);
          tc_after();
          if (elect()) {
#pragma unroll
            for (uint32_t k = part * (Sh::kHalf / 16); k < (part + 1) * (Sh::kHalf / 16); ++k)
              mma_ts<CG>(tm + Sh::kTmemO, tm + buf * KT + k * 8u, d + k * (2048u >> 4), idesc_o, k == 0 ? acc : 1u);
            if (part == 1) {
              tc_commit<CG>(&sh.kv_empty[st]);
              tc_commit<CG>(&sh.pv_done[buf]);
            }
          }
          __syncwarp();
        }
        next_stage();
        if (++pb == NB) pb = 0, pph ^= 1u;
        --left;
      };
      for (; pc.next() && !aborted(sh); pc.advance()) {
        const uint32_t t0 = uniform(pc.t0), t1 = uniform(pc.t1);
        for (uint32_t t = t0; t < t1; ++t, ++g) {
          const uint32_t qb = uniform(job % NQ), buf = uniform(sb);
          if (t == t0) {
            if constexpr (Sh::kDrain)
              while (left) pv();
            wait(sh, &sh.q_full[qb], (job / NQ) & 1u);
          }
          const uint64_t qd = smem_desc(qs + qb * Sh::kQBytes, 16), d = smem_desc(kvs + uniform(st) * Sh::kStageBytes, 16);
          wait(sh, &sh.kv_full[st], ph);
          if (elect()) {
#pragma unroll
            for (uint32_t k = 0; k < D / 16; ++k)
              mma_ss<CG>(tm + buf * KT, qd + ((k >> 2) * kRows * 128u + (k & 3u) * 32u) / 16u,
                         d + ((k >> 2) * Sh::kKeyRows * 128u + (k & 3u) * 32u) / 16u, idesc_s, k > 0);
            tc_commit<CG>(&sh.kv_empty[st]);
            tc_commit<CG>(&sh.s_full[buf]);
            if (t + 1 == t1) tc_commit<CG>(&sh.q_empty[qb]);
          }
          __syncwarp();
          next_stage();
          if (++sb == NB) sb = 0;
          if (left == Sh::kAhead) pv();
#pragma unroll
          for (uint32_t i = Sh::kAhead - 1; i > 0; --i) last[i] = last[i - 1];
          last[0] = Tile{t == t0, pc.keys - t * KT < KT, job};
          ++left;
        }
        if (t1 > t0) ++job;
      }
      while (left && !aborted(sh)) pv();
    } else if (warp == kSoftmaxWarps + 2) {
      // ---- V rows that no query row sees count with weight 0, but 0 times what stands there may be NaN: they are
      // cleared. And a pair's second CTA tells the leader what has landed.
      uint32_t st = 0, ph = 0, jobs = 0, tails = 0, left = 0;
      uint32_t last[Sh::kAhead];  // keys of the tiles whose V is still to come
      auto next_stage = [&] {
        if (++st == ST) st = 0, ph ^= 1u;
      };
      auto v_stage = [&] {
        const uint32_t valid = left == 1 ? last[0] : last[Sh::kAhead - 1];
        // the second CTA's stage waits for its word, the leader's only where the multiplying thread asked for it
        if (rank) wait(sh, &sh.kv_full[st], ph);
        else if (valid < KT) wait(sh, &sh.v_dirty, tails++ & 1u);
        if (valid < KT) {
          const uint32_t base = kv_smem + st * Sh::kStageBytes + lane * 16u;
#pragma unroll 4
          for (uint32_t r = valid; r < KT; r += 4) {  // four rows of 128 bytes at a time
            if (r + lane / 8u < KT) {
#pragma unroll
              for (uint32_t ch = 0; ch < Sh::kVChunks; ++ch)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(base + (ch * KT + r) * 128u), "r"(0u) : "memory");
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          if (rank) asm volatile("fence.acq_rel.cluster;" ::: "memory");
          __syncwarp();
          if (lane == 0 && rank == 0) bar_arrive(&sh.v_clean);
        }
        if (lane == 0 && rank) bar_arrive_leader(&sh.kv_full[st]);
        __syncwarp();
        next_stage();
        --left;
      };
      for (; pc.next() && !aborted(sh); pc.advance()) {
        for (uint32_t t = pc.t0; t < pc.t1; ++t) {
          if (t == pc.t0) {
            if constexpr (Sh::kDrain)
              while (left) v_stage();
            if (rank) {
              wait(sh, &sh.q_full[jobs % NQ], (jobs / NQ) & 1u);
              if (lane == 0) bar_arrive_leader(&sh.q_full[jobs % NQ]);
              ++jobs;
            }
          }
          if (rank) {
            wait(sh, &sh.kv_full[st], ph);
            if (lane == 0) bar_arrive_leader(&sh.kv_full[st]);
            __syncwarp();
          }
          next_stage();
          if (left == Sh::kAhead) v_stage();
#pragma unroll
          for (uint32_t i = Sh::kAhead - 1; i > 0; --i) last[i] = last[i - 1];
          last[0] = min(KT, pc.keys - t * KT);
          ++left;
        }
      }
      while (left && !aborted(sh)) v_stage();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    Pieces<KT> pc(c, sh, tq);
    auto tell_leader = [&](unsigned long long* b) {
      if (rank == 0) bar_arrive(b);
      else bar_arrive_leader(b);
    };
    // ---- softmax, and the outputs -------------------------------------------------------------------------------
    constexpr uint32_t HK = Sh::kHalf;
    const uint32_t pair = warp >> 3, half = (warp >> 2) & 1u, quad = warp & 3u, row = quad * 32u + lane;
    const uint32_t lane_base = (quad * 32u) << 16;
    const uint32_t my_tok = row / c.group, my_head = row - my_tok * c.group;
    // the 64 threads of a pair that share 32 rows
    auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1u + pair * 4u + quad) : "memory"); };
    uint32_t g = 0, job = 0;  // tiles so far, pieces with tiles
    if (threadIdx.x == 0 && rank == 0) c.meta[8u * unit] = c.meta[8u * unit + 1] = 0;
    for (; pc.next(); pc.advance()) {
      const uint32_t tok0 = pc.i * tq + rank * tq_cta;
      const uint32_t rows = tok0 < pc.s.rows ? min(tq_cta, pc.s.rows - tok0) * c.group : 0u;  // of this CTA
      const bool busy = quad * 32u < rows;  // warps without a row only keep step
      // keys that this row sees
      uint32_t limit = pc.keys;
      if (c.causal) limit = static_cast<uint32_t>(max(0, min(static_cast<int>(pc.keys), pc.s.off + static_cast<int>(tok0 + my_tok) + 1)));
      const uint32_t all_see = c.causal ? static_cast<uint32_t>(max(0, pc.s.off + static_cast<int>(tok0) + 1)) : pc.keys;
      float m = -INFINITY, l = 0.0f;  // the reference that l is relative to
      float before = -INFINITY;       // the one of the tile before
      const uint32_t g0 = g;
      g += pc.t1 - pc.t0;
      for (uint32_t t = pc.t0 + ((g0 ^ pair) & 1u); t < pc.t1; t += 2) {
        const uint32_t g = g0 + (t - pc.t0);
        const uint32_t buf = g % NB, slot = g % NS;
        wait(sh, &sh.s_full[buf], (g / NB) & 1u);
        tc_after();
        if (busy) {
          float s[HK / 32][32];
#pragma unroll
          for (uint32_t x = 0; x < HK / 32; ++x) tc_ld32(tmem + lane_base + buf * KT + half * HK + x * 32u, s[x]);
          float ref = -INFINITY;  // the other pair's, of the tile before
          if (half == 0 && t > pc.t0) {
            wait(sh, &sh.m_full[(g - 1) % NS][quad], ((g - 1) / NS) & 1u);
            ref = sh.m[(g - 1) % NS][row];
          }
          tc_wait_ld(s);
          const uint32_t key0 = t * KT + half * HK;
          if (key0 + HK > min(all_see, pc.keys)) {
            const uint32_t left = limit > key0 ? limit - key0 : 0u;
#pragma unroll
            for (uint32_t x = 0; x < HK / 32; ++x) {
              const uint32_t over = left > x * 32 ? left - x * 32 : 0u, keep = over >= 32 ? 0xFFFFFFFFu : (1u << over) - 1u;
#pragma unroll
              for (uint32_t y = 0; y < 32; ++y)
                if (!(keep & (1u << y))) s[x][y] = -INFINITY;
            }
          }
          float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains
#pragma unroll
          for (uint32_t x = 0; x < HK; x += 2) part[x / 2 % 4] = max3f(part[x / 2 % 4], s[x / 32][x % 32], s[x / 32][x % 32 + 1]);
          float mx = fmaxf(max3f(part[0], part[1], part[2]), part[3]);
          if (row >= rows) mx = -INFINITY;  // no query row: what stands there has no say
          trade_maxima(sh.trade[pair][trade_of(g)], half, row, mx, ref, [&] {
            tc_before();  // behind this P of either group may replace S
            pair_sync();
            tc_after();
          });
          before = ref;
          // the reference follows where it has fallen too far behind
          const float grown = __fmul_rn(mx - ref, c.scale_log2);
          const bool follow = grown > kLazy;  // also from -inf; false for -inf against -inf (NaN)
          float next_ref = follow ? mx : ref;
          if (__any_sync(kFullMask, follow && ref != -INFINITY)) {  // in both groups of the pair alike
            wait(sh, &sh.pv_done[(g - 1) % NB], ((g - 1) / NB) & 1u);
            tc_after();
            const float f = follow && ref != -INFINITY ? ex2_approx(-grown) : 1.0f;
#pragma unroll 1
            for (uint32_t x = 0; x < D / 2; x += 16) {
              uint32_t o[16];
              tc_ld16(tmem + lane_base + Sh::kTmemO + half * (D / 2) + x, o);
              tc_wait_ld16(o);
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__fmul_rn(__uint_as_float(o[y]), f));
              tc_st16(tmem + lane_base + Sh::kTmemO + half * (D / 2) + x, o);
            }
            tc_wait_st();
            tc_before();
            pair_sync();  // the first part of P is handed on when all columns are done
            tc_after();
          }
          if (half == 0) {
            sh.m[slot][row] = next_ref;
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.m_full[slot][quad]);
            // The other pair waits for that. Reading the reference back makes the exponentials depend on it; without that the
            // assembler puts the arrival behind them, and the pairs take turns instead of overlapping (1900 instead of
            // 1400 cycles a tile at D = 64).
            next_ref = *static_cast<volatile float*>(&sh.m[slot][row]);
          }
          // p = 2^(c s - c ref); a row that has seen nothing yet has s = -inf everywhere, and 0 does for its reference
          const float mc = next_ref == -INFINITY ? 0.0f : __fmul_rn(next_ref, c.scale_log2);
          const float2 c2 = make_float2(c.scale_log2, c.scale_log2), m2 = make_float2(kLift<T> - mc, kLift<T> - mc);
          float2 sum[2] = {};
          uint32_t r[HK / 2];
#pragma unroll
          for (uint32_t y = 0; y < HK / 2; ++y) {
            const uint32_t at = 2 * y;
            float2 v = __ffma2_rn(make_float2(s[at / 32][at % 32], s[at / 32][at % 32 + 1]), c2, m2);
            v.x = ex2_approx(v.x);
            v.y = ex2_approx(v.y);
            sum[y % 2] = __fadd2_rn(sum[y % 2], v);
            r[y] = pack2<T>(v.x, v.y);
          }
          if constexpr (HK == 64) tc_st32(tmem + lane_base + buf * KT + half * (HK / 2), r);
          else tc_st16(tmem + lane_base + buf * KT + half * (HK / 2), r);
          if (next_ref != m) {
            if (m != -INFINITY) l = __fmul_rn(l, ex2_approx(__fmul_rn(m - next_ref, c.scale_log2)));
            m = next_ref;
          }
          sum[0] = __fadd2_rn(sum[0], sum[1]);
          l += sum[0].x + sum[0].y;
          tc_wait_st();
        } else if (half == 0 && lane == 0) {
          bar_arrive(&sh.m_full[slot][quad]);
        }
        tc_before();
        __syncwarp();
        if (lane == 0) tell_leader(&sh.p_full[buf][half]);
      }
      const bool any = pc.t1 > pc.t0, whole = pc.t0 == 0 && pc.t1 == pc.n;
      // The pair of the last tile writes the outputs, while the other one, having left its denominator behind, goes on
      // to the next job's first tile. (No pair is NS jobs ahead of the other: O takes the products of one job at a time.)
      const bool owner = any ? ((g - 1) & 1u) == pair : pair == 0;
      float* sl = &sh.l[job % NS][row];
      unsigned long long* l_full = &sh.l_full[job % NS][quad];
      const uint32_t l_phase = (job / NS) & 1u;
      if (any) ++job;
      if (!owner) {
        if (any) {
          if (half == 1) *sl = l;
          pair_sync();
          if (half == 0) {
            *sl += l;
            __syncwarp();
            if (lane == 0) bar_arrive(l_full);
          }
        }
      } else {
        const float ref = m;
        float total = 0.0f;
        if (any) {
          wait(sh, l_full, l_phase);
          // over the reference of the tile before the last one; without one it is 0, or NaN from scores that are NaN
          const float other = *sl, others = before == ref || before == -INFINITY
                                                ? other
                                                : __fmul_rn(other, ex2_approx(__fmul_rn(before - ref, c.scale_log2)));
          pair_sync();
          if (half == 1) *sl = l;
          pair_sync();
          if (half == 0) *sl = (l + *sl) + others;
          pair_sync();
          total = *sl;
        }
        if (any) {
          wait(sh, &sh.pv_done[(g - 1) % NB], ((g - 1) / NB) & 1u);
          tc_after();
        }
        const bool mine = row < rows && !aborted(sh);
        const uint64_t token = pc.s.row0 + tok0 + my_tok;
        const uint32_t head = pc.h * c.group + my_head;
        const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
        if (busy && whole) {
          T* out4[4];  // where the rows of this lane's four go; null: no row
          T* to = mine ? static_cast<T*>(c.out) + token * c.out_row + head * c.out_head : nullptr;
#pragma unroll
          for (uint32_t y = 0; y < 4; ++y)
            out4[y] = reinterpret_cast<T*>(__shfl_sync(kFullMask, reinterpret_cast<unsigned long long>(to), (lane & ~3u) + y));
          // The loop stays rolled: unrolled, its first pass is bound by instruction fetches (10000 cycles for 64 KB).
#pragma unroll 1
          for (uint32_t x = half * (D / 2); x < (half + 1) * (D / 2); x += 32) {
            float o[32];
            tc_ld32(tmem + lane_base + Sh::kTmemO + x, o);
            tc_wait_ld(o);
            uint4 u[4];
#pragma unroll
            for (uint32_t y = 0; y < 4; ++y) {
              u[y].x = pack2<T>(__fmul_rn(o[8 * y], inv), __fmul_rn(o[8 * y + 1], inv));
              u[y].y = pack2<T>(__fmul_rn(o[8 * y + 2], inv), __fmul_rn(o[8 * y + 3], inv));
              u[y].z = pack2<T>(__fmul_rn(o[8 * y + 4], inv), __fmul_rn(o[8 * y + 5], inv));
              u[y].w = pack2<T>(__fmul_rn(o[8 * y + 6], inv), __fmul_rn(o[8 * y + 7], inv));
              if (total == 0.0f) u[y] = make_uint4(0, 0, 0, 0);  // no key (and without tiles O holds anything)
            }
            // A lane holds 64 bytes of its own row; a store of those would touch 32 lines. Four lanes trade their four
            // 16-byte parts, so that each store covers 64 bytes of each of eight rows.
            trade4(u, lane);
            const uint32_t at = x + (lane & 3u) * 8u;
            if (at < c.dim) {
#pragma unroll
              for (uint32_t y = 0; y < 4; ++y)
                if (out4[y]) *reinterpret_cast<uint4*>(out4[y] + at) = u[y];
            }
          }
          if (mine && c.lse && half == 0)
            c.lse[token * (c.kv_heads * c.group) + head] =
                total == 0.0f ? -INFINITY : __fmul_rn(__fmaf_rn(ref, c.scale_log2, __log2f(total) - kLift<T>), 0.69314718055994531f);
        } else if (busy) {  // a piece of a split job; pieces have tiles
          float* piece = c.part + ((2ull * unit + (pc.t0 == 0 ? 1u : 0u)) * CG + rank) * AttnPieceFloats(D);
#pragma unroll 1
          for (uint32_t x = half * (D / 2); x < (half + 1) * (D / 2); x += 32) {
            float o[32];
            tc_ld32(tmem + lane_base + Sh::kTmemO + x, o);
            tc_wait_ld(o);
            // [column / 4][row] quads, so that a warp's rows lie side by side
            if (mine) {
#pragma unroll
              for (uint32_t y = 0; y < 32; y += 4)
                *reinterpret_cast<float4*>(piece + ((x + y) / 4 * kRows + row) * 4) = make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]);
            }
          }
          if (mine && half == 0) {
            piece[D * kRows + row] = ref;
            piece[(D + 1) * kRows + row] = total;
          }
        }
        tc_before();
        __syncwarp();
        if (any && lane == 0) tell_leader(&sh.o_empty);
      }
      if (threadIdx.x == 0 && rank == 0 && !whole) {
        // what the join needs: a piece that opens a split job says which one, every other one whether it ends it
        uint32_t* to = c.meta + 8u * unit;
        if (pc.t0 == 0) to[1] = 1u, to[2] = pc.s.row0 + pc.i * tq, to[3] = min(tq, pc.s.rows - pc.i * tq), to[4] = pc.h;
        else to[0] = pc.t1 == pc.n ? 2u : 1u;
      }
    }
  }

  __syncwarp();
  if constexpr (CG == 2) {  // a pair's CTAs end alike: the products use the operands and barriers of both
    if (lane == 0 && aborted(sh))
      asm volatile("{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %0, %1;\nst.shared::cluster.u32 [r], %2;\n}" ::"r"(smem_addr(&sh.abort)),
                   "r"(rank ^ 1u), "r"(1u)
                   : "memory");
    __syncwarp();
  }
  tc_before();
  sync_all<CG>();
  tc_after();
  if (aborted(sh)) {  // nobody waits any more, so all threads of both CTAs see the same
    if (warp == kSoftmaxWarps + 1 && rank == 0 && elect()) tc_commit<CG>(&sh.drained);
    if (threadIdx.x == 0) stage_wait(smem_addr(&sh.drained), 0);
    __syncwarp();
    sync_all<CG>();
  }
  if (warp == kSoftmaxWarps + 1) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}


// ---- joining the pieces of split jobs -----------------------------------------------------------------------------
// out = sum_p 2^(c (r_p - R)) O_p / sum_p 2^(c (r_p - R)) l_p over a job's pieces p, R the largest of their references.
// blockIdx.x: the split job, counted over the units that opened one; blockIdx.y: 32 rows (lane = row) and a share of the
// columns. What bounds it is latency: a chain of dependent round trips to L2 (flags, then everything else), so all loads
// of a stage are in flight together. Few pieces (a prompt's jobs are cut once): a warp sums its column quads over all
// of them and keeps the weights in registers. Many (one token over a long cache is cut by every unit): the warps share
// the pieces and meet in shared memory. The order of the sums is fixed.
constexpr uint32_t kJoinResident = 4;  // CTAs on an SM: a grid of one wave (in four waves of two the join of 74 jobs took 17 us)
constexpr uint32_t kJoinWarps = 8, kFew = 4, kFewQuads = 4, kManyQuads = 2;
template <typename T, int D, int CG>
__global__ void __launch_bounds__(kJoinWarps * 32, kJoinResident) attention_join_kernel(const __grid_constant__ AttnCall c, const uint32_t units) {
  constexpr uint32_t kWords = (kMaxCtas + 31) / 32;
  __shared__ uint32_t opens[kWords], ends[kWords];
  __shared__ float meet[kJoinWarps][32];
  __shared__ float4 red[kJoinWarps][kManyQuads][32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  pdl_wait_and_trigger();
  if (warp < kWords) {
    const uint32_t x = warp * 32u + lane;
    const uint2 f = x < units ? *reinterpret_cast<const uint2*>(c.meta + 8u * x) : make_uint2(0, 0);
    const uint32_t o = __ballot_sync(kFullMask, f.y == 1u), e = __ballot_sync(kFullMask, f.x == 2u);
    if (lane == 0) opens[warp] = o, ends[warp] = e;
  }
  __syncthreads();
  uint32_t k = blockIdx.x, first = kMaxCtas;
  for (uint32_t w = 0; w < kWords; ++w) {
    const uint32_t n = __popc(opens[w]);
    if (k < n) {
      uint32_t v = opens[w];
      for (; k; --k) v &= v - 1;
      first = w * 32u + __ffs(v) - 1;
      break;
    }
    k -= n;
  }
  if (first >= units) return;
  uint32_t last = first;
  for (uint32_t w = (first + 1) / 32; w < kWords; ++w) {
    uint32_t v = ends[w];
    if (w == (first + 1) / 32) v &= ~0u << ((first + 1) & 31u);
    if (v) {
      last = w * 32u + __ffs(v) - 1;
      break;
    }
  }
  const uint32_t pieces = last - first + 1;
  // the first rows' blocks are the first of the grid: of a single token's tile no others have work
  const uint32_t parts = gridDim.y / (4 * CG), group = blockIdx.y / parts, rank = group >> 2, row = (group & 3u) * 32u + lane;
  // piece 0 opened the job, the others are what the units behind began with
  auto piece = [&](uint32_t p) { return c.part + ((2ull * (first + p) + (p == 0 ? 1u : 0u)) * CG + rank) * AttnPieceFloats(D); };
  const uint4 job = *reinterpret_cast<const uint4*>(c.meta + 8u * first);  // ., ., first token, tokens
  const uint32_t h = c.meta[8u * first + 4];
  const uint32_t tq_cta = kRows / c.group, tok0 = rank * tq_cta;
  const uint32_t rows = tok0 < job.w ? min(tq_cta, job.w - tok0) * c.group : 0u;
  if ((group & 3u) * 32u >= rows) return;
  const bool mine = row < rows;
  const uint64_t token = job.z + tok0 + row / c.group;
  const uint32_t head = h * c.group + row % c.group;
  T* out = static_cast<T*>(c.out) + token * c.out_row + head * c.out_head;
  const uint32_t quads = D / 4 / parts, q0 = (blockIdx.y - group * parts) * quads;
  auto finish2 = [&](uint32_t q, const float4 (&sum)[2], float inv) {  // two quads, q even
    if (mine && q * 4 < c.dim) {
      uint4 u;
      u.x = pack2<T>(__fmul_rn(sum[0].x, inv), __fmul_rn(sum[0].y, inv));
      u.y = pack2<T>(__fmul_rn(sum[0].z, inv), __fmul_rn(sum[0].w, inv));
      u.z = pack2<T>(__fmul_rn(sum[1].x, inv), __fmul_rn(sum[1].y, inv));
      u.w = pack2<T>(__fmul_rn(sum[1].z, inv), __fmul_rn(sum[1].w, inv));
      *reinterpret_cast<uint4*>(out + q * 4) = u;
    }
  };
  auto finish_lse = [&](float top, float total) {
    if (c.lse && q0 == 0 && warp == 0 && mine)
      c.lse[token * (c.kv_heads * c.group) + head] =
          total == 0.0f ? -INFINITY : __fmul_rn(__fmaf_rn(top, c.scale_log2, __log2f(total) - kLift<T>), 0.69314718055994531f);
  };
  // A piece without a maximum has no weight (-1): its sums say nothing. Its denominator does: 0, or NaN where its scores were
  // NaN, which has no part in a maximum. A NaN denominator, behind a weight of 0 too, makes the joined one and so all outputs NaN.
  auto add = [](float4& sum, float w, float4 v) {
    if (!(w < 0.0f)) {
      sum.x = __fmaf_rn(w, v.x, sum.x);
      sum.y = __fmaf_rn(w, v.y, sum.y);
      sum.z = __fmaf_rn(w, v.z, sum.z);
      sum.w = __fmaf_rn(w, v.w, sum.w);
    }
  };
  auto quad = [&](uint32_t p, uint32_t q) { return *reinterpret_cast<const float4*>(piece(p) + (q * kRows + row) * 4); };
  auto weight = [&](float r, float top) { return r == -INFINITY ? -1.0f : ex2_approx(__fmul_rn(r - top, c.scale_log2)); };

  if (pieces <= kFew) {
    float r[kFew], l[kFew], top = -INFINITY, total = 0.0f;
#pragma unroll
    for (uint32_t p = 0; p < kFew; ++p) {
      r[p] = mine && p < pieces ? piece(p)[D * kRows + row] : -INFINITY;
      l[p] = mine && p < pieces ? piece(p)[(D + 1) * kRows + row] : 0.0f;
    }
    // Two pieces are by far the most common: their loads do not wait for the weights. A warp takes four neighbouring
    // quads, so that a lane's 16 values fill a 32-byte sector of the output.
    for (uint32_t q = q0 + warp * kFewQuads; q < q0 + quads; q += kJoinWarps * kFewQuads) {
      float4 v[2][kFewQuads];
#pragma unroll
      for (uint32_t x = 0; x < kFewQuads; ++x)
#pragma unroll
        for (uint32_t p = 0; p < 2; ++p) v[p][x] = mine ? quad(p, q + x) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (q == q0 + warp * kFewQuads) {
#pragma unroll
        for (uint32_t p = 0; p < kFew; ++p) top = fmaxf(top, r[p]);
#pragma unroll
        for (uint32_t p = 0; p < kFew; ++p) {
          r[p] = weight(r[p], top);
          total = __fmaf_rn(fabsf(r[p]), l[p], total);
        }
      }
      const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
#pragma unroll
      for (uint32_t x = 0; x < kFewQuads; x += 2) {
        float4 sum[2] = {};
#pragma unroll
        for (uint32_t y = 0; y < 2; ++y) {
          add(sum[y], r[0], v[0][x + y]);
          add(sum[y], r[1], v[1][x + y]);
          if (mine && pieces > 2) add(sum[y], r[2], quad(2, q + x + y));
          if (mine && pieces > 3) add(sum[y], r[3], quad(3, q + x + y));
        }
        finish2(q + x, sum, inv);
      }
    }
    finish_lse(top, total);
    return;
  }

  // each warp over its pieces, then all warps over the warps
  auto ref = [&](uint32_t p) { return mine ? piece(p)[D * kRows + row] : -INFINITY; };
  float top = -INFINITY, total = 0.0f;
#pragma unroll 4
  for (uint32_t p = warp; p < pieces; p += kJoinWarps) top = fmaxf(top, ref(p));
  meet[warp][lane] = top;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < kJoinWarps; ++w) top = fmaxf(top, meet[w][lane]);
  __syncthreads();
#pragma unroll 4
  for (uint32_t p = warp; p < pieces; p += kJoinWarps) {
    const float l = mine ? piece(p)[(D + 1) * kRows + row] : 0.0f;
    total = __fmaf_rn(fabsf(weight(ref(p), top)), l, total);
  }
  meet[warp][lane] = total;
  __syncthreads();
  total = 0.0f;
#pragma unroll
  for (uint32_t w = 0; w < kJoinWarps; ++w) total += meet[w][lane];
  const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
  finish_lse(top, total);
  for (uint32_t q = q0; q < q0 + quads; q += kManyQuads) {
    float4 sum[kManyQuads] = {};
    if (mine) {
#pragma unroll 3
      for (uint32_t p = warp; p < pieces; p += kJoinWarps) {
        const float w = weight(ref(p), top);
#pragma unroll
        for (uint32_t x = 0; x < kManyQuads; ++x) add(sum[x], w, quad(p, q + x));
      }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t x = 0; x < kManyQuads; ++x) red[warp][x][lane] = sum[x];
    __syncthreads();
    if (warp == 0) {
      float4 all[2] = {};
#pragma unroll
      for (uint32_t w = 0; w < kJoinWarps; ++w)
#pragma unroll
        for (uint32_t x = 0; x < 2; ++x) {
          const float4 v = red[w][x][lane];
          all[x].x += v.x, all[x].y += v.y, all[x].z += v.z, all[x].w += v.w;
        }
      finish2(q, all, inv);
    }
  }
}

// ---- launch -----------------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn Encoder() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// A map over 16-bit elements with 128-byte swizzle; dims[0] is contiguous, strides in elements. The stride of an axis
// with one entry is never used, but has to pass the encoder's checks.
cudaError_t MakeMap(CUtensorMap* map, int dtype, const void* base, uint32_t rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box) {
  const EncodeFn encode = Encoder();
  if (!encode) return cudaErrorNotSupported;
  cuuint64_t d[4], st[3];
  cuuint32_t b[4], es[4] = {1, 1, 1, 1};
  for (uint32_t i = 0; i < rank; ++i) d[i] = dims[i], b[i] = box[i];
  for (uint32_t i = 1; i < rank; ++i) st[i - 1] = dims[i] == 1 ? 16 * ((dims[0] * 2 + 15) / 16) : strides[i] * 2;
  const CUresult r = encode(map, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base), d,
                            st, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

constexpr uint64_t kMetaBytes = 8192;
static_assert(kMetaBytes >= kMaxCtas * 32, "eight words for each CTA");
constexpr uint32_t PadDim(uint32_t dim) { return dim <= 64 ? 64u : dim <= 128 ? 128u : 256u; }

template <typename T, int D, int CG>
cudaError_t Launch(const AttnArgs& a, cudaStream_t s) {
  AttnCall c{};
  c.cu = a.cu;
  c.kv_len = a.kv_len;
  c.table = a.table;
  c.table_stride = a.table_stride;
  c.table_cols = a.table_cols;
  c.page_shift = a.page_shift;
  c.batch = a.batch;
  c.tokens = a.tokens;
  c.kv_heads = a.kv_heads;
  c.group = a.q_heads / a.kv_heads;
  c.dim = a.dim;
  c.causal = a.causal;
  c.scale_log2 = static_cast<float>(static_cast<double>(a.scale) * 1.4426950408889634);
  c.out = a.out;
  c.out_row = a.out_row;
  c.out_head = a.out_head;
  c.lse = a.lse;
  c.meta = static_cast<uint32_t*>(a.workspace);
  c.part = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + kMetaBytes);
  const uint32_t tq_cta = kRows / c.group, tq = CG * tq_cta;
  c.box_shift = a.table && a.page_shift < 6u ? a.page_shift : 6u;

  CUtensorMap qm, km, vm;
  const uint64_t qd[3] = {a.dim, a.q_heads, a.tokens}, qs[3] = {1, a.q_head, a.q_row};
  const uint32_t qb[3] = {64, c.group, tq_cta};
  cudaError_t e = MakeMap(&qm, a.dtype, a.q, 3, qd, qs, qb);
  if (e != cudaSuccess) return e;
  const uint64_t rows = a.table ? uint64_t{1} << a.page_shift : a.tokens, pages = a.table ? a.pages : 1;
  const uint64_t kd[4] = {a.dim, rows, a.kv_heads, pages};
  const uint64_t ks[4] = {1, a.k_row, a.k_head, a.k_page}, vs[4] = {1, a.v_row, a.v_head, a.v_page};
  const uint32_t kb[4] = {64, 1u << c.box_shift, 1, 1};
  e = MakeMap(&km, a.dtype, a.k, 4, kd, ks, kb);
  if (e == cudaSuccess) e = MakeMap(&vm, a.dtype, a.v, 4, kd, vs, kb);
  if (e != cudaSuccess) return e;

  int dev = 0, sms = 0;
  e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(attention_kernel<T, D, CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes<D, CG>));
  if (e != cudaSuccess) return e;
  // setmaxnreg hands on what the launch has: with fewer registers a thread than the shares were added up for, the softmax
  // groups would wait for good
  static std::atomic<bool> checked{false};
  if (!checked.load(std::memory_order_relaxed)) {
    cudaFuncAttributes f;
    e = cudaFuncGetAttributes(&f, attention_kernel<T, D, CG>);
    if (e != cudaSuccess) return e;
    if (f.numRegs != static_cast<int>(kLaunchRegs)) return cudaErrorInvalidConfiguration;
    checked.store(true, std::memory_order_relaxed);
  }
  const uint64_t most_keys = a.table ? static_cast<uint64_t>(a.table_cols) << a.page_shift : a.tokens;
  const uint64_t jobs = (static_cast<uint64_t>(a.tokens) / tq + a.batch) * a.kv_heads;  // at most
  const uint64_t tiles = (most_keys + Shape<D, CG>::kKeys - 1) / Shape<D, CG>::kKeys;
  uint64_t units = (jobs * (tiles + kJobCost) + kMinShare - 1) / kMinShare;
  const uint64_t most_units = static_cast<uint64_t>(sms < static_cast<int>(kMaxCtas) ? sms : static_cast<int>(kMaxCtas)) / CG;
  if (units > most_units) units = most_units;
  if (units < 1) units = 1;

  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = static_cast<unsigned>(units * CG);
  cfg.blockDim = kThreads;
  cfg.dynamicSmemBytes = kSmemBytes<D, CG>;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PdlEnabled() ? 2u : 1u;
  e = cudaLaunchKernelEx(&cfg, attention_kernel<T, D, CG>, c, qm, km, vm);
  // jobs of one tile are never split
  if (e != cudaSuccess || tiles <= 1 || units == 1) return e;
  const uint32_t x = static_cast<uint32_t>(jobs < units ? jobs : units);
  // one wave of blocks with work: a pair's tiles are mostly full, a single CTA's mostly hold 32 rows at most
  const uint32_t groups = CG == 2 ? 8 : 1;
  uint32_t parts = 1;
  while (parts < D / 16 && x * groups * parts * 2 <= static_cast<uint32_t>(sms) * kJoinResident) parts *= 2;
  return LaunchKernel(attention_join_kernel<T, D, CG>, dim3(x, 4 * CG * parts), kJoinWarps * 32, 0, s, c, static_cast<uint32_t>(units));
}

// A pair's tile has twice the rows, and half of it is idle where a sequence's rows (tokens x heads of a group) do not fill
// it: pairs from three CTAs' rows a sequence on. Measured, single CTA against pair, 8 sequences behind 4096 keys, 16/2 heads
// of 256: 64 rows 26 / 50 us, 128 rows 34 / 45, 192 rows 40 / 45, 384 rows 47 / 48 (heads of 128: 33.5 / 32); one prompt of 4096
// tokens 146 / 116; 8 single tokens over 2 GB 312 / 372.
template <typename T, int D>
cudaError_t LaunchPair(const AttnArgs& a, cudaStream_t s) {
  if (static_cast<uint64_t>(a.tokens) * (a.q_heads / a.kv_heads) >= static_cast<uint64_t>(a.batch) * (3 * kRows)) return Launch<T, D, 2>(a, s);
  return Launch<T, D, 1>(a, s);
}

template <typename T>
cudaError_t LaunchDim(const AttnArgs& a, cudaStream_t s) {
  switch (PadDim(a.dim)) {
    // no pair at 64: its second CTA would stage half of V's columns, and 64 of them are one 128-byte swizzled chunk
    case 64: return Launch<T, 64, 1>(a, s);
    case 128: return LaunchPair<T, 128>(a, s);
    default: return LaunchPair<T, 256>(a, s);
  }
}

}  // namespace

uint64_t AttentionWorkspaceBytes(uint32_t dim) { return kMetaBytes + 2ull * kMaxCtas * AttnPieceFloats(PadDim(dim)) * 4; }

cudaError_t LaunchAttention(const AttnArgs& a, cudaStream_t s) {
  return a.dtype == kBF16 ? LaunchDim<bf16>(a, s) : LaunchDim<f16>(a, s);
}

cudaError_t ReadAttentionTimeouts(unsigned int* out) { return cudaMemcpyFromSymbol(out, g_attn_timeouts, sizeof(unsigned int)); }

}  // namespace halo_b200
