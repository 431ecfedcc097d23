// Linear attention by chunks of 128 tokens on the tensor cores (see linear_attention.cuh for what a
// pass computes).  Within a chunk, with i and j its tokens, w the decays between them and S the state
// before it,
//   scores = A B^T,   P = scores . w (0 where j is later than i),
//   O = scale * (P C + e^(g (i + 1)) (A S)),   S <- e^(g 128) S + (left . B)^T C
// (left: the decay from a token to the chunk's end).  Four products of 128 x 128 x 128, the last in two
// or three parts, per chunk of four 32 KiB tiles read or written: 160 flop per byte, so HBM would be the
// bound, 3.0 us a chunk when 148 blocks share the measured bandwidth.  The work of a chunk is a chain,
// scores (760 cycles) -> P (2400) -> P C (1050) -> the state (1050) -> its copy, of which the tiles'
// loads, left . B, the next scores and the output run beside: 5300 cycles a chunk of 128 channels, 4100 of
// 64, 2.7 us at 1965 MHz (8 sequences of 2048 tokens x 64 heads x 128: 226 to 240 us after a rest, HBM 164).
// In long loops the power limit holds the clock at 1.43 to 1.5 GHz and the same takes 276 to 293 us.  (The
// state's product reads nothing of P: it stands in the chain only because it is issued after P C.  The other
// order has not been tried.)
// Measured level or slower, and not kept: P by eight warps, A in TMEM, the output by way of shared memory
// and TMA, P C begun on the first half of P (0-2 %, more spills), the moves of states shared with the warps
// of left . B; one part of left . B instead of two would save 3 %.
//
// One block per SM walks (sequence, head) pairs with 768 threads:
//   warp 0       TMA producer: tiles of A, B and C, 128 tokens x 64 channels a box, 128-byte swizzle.
//   warp 1       MMA issuer.  TMEM, 128 columns each: scores and P, A S, P C, and the state in FP32.
//   warps 2-3    infinities and NaN in C (below).
//   warps 4-7    scores -> P (BF16, back into TMEM as the A operand of P C).
//   warps 8-15   the output.
//   warps 16-19  the state: its BF16 copy in shared memory for A S, and its decay in TMEM.
//   warps 20-23  left . B.
// Roundings: P and the copy of S are BF16, as operands have to be; the state itself stays FP32.  Where the
// chunks are not more than the SMs, or sequences have four tokens or fewer on average (kFine), P is two
// BF16 parts, its sum to 2^-17: few scores' roundings do not average out (a token's output could be 2^-8
// off).  The time is small beside a launch's (4096 tokens of one head 39 us, 37 with one part; 37 tokens
// of 16 heads no difference), but not with many short sequences (64 of 4 tokens x 32 heads 84 us, 66).  left . B
// is split into BF16 parts whose sum it is to 2^-17 (two products), or, where the state is an output
// (kExact), to 2^-25 (three).  The tensor cores cut off a sum's last bits every 16 tokens: 24 times a
// chunk at the state's size would leave it 1e-6 off.  The two small parts are summed apart then, in P's
// columns, and added in FP32: 2e-7, as with FP32 throughout (8 sequences of 2048 x 64 heads x 128 with
// final states in a loop: 350 us, 321 in one sum, 277 without final states).
// An infinity or NaN in C would spoil its channel in all of the chunk's outputs, the earlier ones too
// (0 times it is NaN).  It is replaced by 0, and its channel is NaN from its token on in what is
// written.
#pragma once
#include "linear_attention.cuh"
#include "ptx.cuh"

namespace cpg {

constexpr int kChunk = 128;
constexpr int kChunkThreads = 768;

// Wait sites (low byte of the status word).
enum : int32_t {
  kSiteLinearProducer = 0x60,
  kSiteLinearMma = 0x61,
  kSiteLinearScores = 0x62,
  kSiteLinearState = 0x63,
  kSiteLinearOutput = 0x64,
  kSiteLinearLeft = 0x65,
  kSiteLinearScan = 0x66,
  kSiteLinearDrain = 0x67,
};

constexpr uint64_t kLinearDrainNs = 100000000;

// Host-selected, for testing the bounded waits: the producer loads nothing, or no tile of C.
constexpr int32_t kLinearSkipLoads = 1, kLinearSkipValues = 2;

// First error of any launch on this device (0: none).
__device__ int32_t linear_status_word;

template <int DA, int DC>
struct ChunkLayout {
  static constexpr uint32_t kTileA = kChunk * DA * 2;  // also of B and its parts
  static constexpr uint32_t kTileC = kChunk * DC * 2;
  static constexpr uint32_t kTileS = DA * DC * 2;
  static constexpr uint32_t kA = 0;
  static constexpr uint32_t kB = kA + kTileA;          // 2 slots
  static constexpr uint32_t kMid = kB + 2 * kTileA;    // second part of left . B
  static constexpr uint32_t kC = kMid + kTileA;        // 2 slots
  // Third part: a tile of its own, or where there is no room for one C's second slot, so that C has
  // one then.  (The state's product takes 128 rows of a part even where B has 64 channels: its second
  // 64, rows of the result that nothing reads, are whatever lies one box further on, in the next
  // tile.)
  static constexpr bool kShared = DA == 128 && DC == 128;
  static constexpr uint32_t kLo = kShared ? kC + kTileC : kC + 2 * kTileC;
  static constexpr uint32_t kS = kLo + kTileA;
  static constexpr uint32_t kBars = kS + (kTileS > 16384u ? kTileS : 16384u);
  static constexpr uint32_t kNumBars = 22;
  static constexpr uint32_t kSlot = kBars + kNumBars * 8;
  static constexpr uint32_t kPowers = kSlot + 16;      // 64 for each warp of the scores
  static_assert(kPowers % 16 == 0, "read four at a time");
  static constexpr uint32_t kBad = kPowers + 4 * 256;  // of every channel of C, the last of all, progress
  static constexpr uint32_t kBytes = kBad + kChunk * 4 + 64 + 1024;
  static_assert(kBytes <= 232448, "shared memory of a block");
};

// TMEM columns.
constexpr uint32_t kColScores = 0, kColInter = 128, kColIntra = 256, kColState = 384;

// Instruction descriptor of kind::f16 with BF16 operands, FP32 accumulators; a set bit: the operand's
// rows run along the reduction (its M or N channels are contiguous).
__host__ __device__ constexpr uint32_t linear_idesc(int n, bool a_mn, bool b_mn) {
  return ptx::make_idesc_bf16_f32(128, n) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
}

// Low halves of shared-memory descriptors (the high half is the GEMM kernels': rows of 128 bytes,
// 128-byte swizzle, 8-row groups 1024 bytes apart).  For an operand whose rows run along the
// reduction the leading offset is that from one box of 64 channels to the next.
__device__ __forceinline__ uint32_t desc_lo_mn(uint32_t addr, uint32_t box_bytes) {
  return ((addr >> 4) & 0x3FFFu) | (box_bytes >> 4) << 16;
}

// Step k of 16 channels in an operand along its channels (in units of 16 bytes).
__device__ __forceinline__ uint32_t k_step(uint32_t k) { return (k >> 2) * 1024 + (k & 3) * 2; }

// D[tmem] (+)= A * B[smem], A in TMEM or shared memory, issued by the lane whose `issue` is set.  All
// lanes of the warp come here together: descriptors that are the same in each can then be made in
// uniform registers, where the instruction wants them (made by one lane of a divergent warp, they
// took twice the time of the products).
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo,
                                            uint32_t idesc, uint32_t accumulate, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(ptx::sw128_desc_hi()), "r"(idesc), "r"(accumulate), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                            uint32_t idesc, uint32_t accumulate, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(ptx::sw128_desc_hi()), "r"(idesc), "r"(accumulate), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint32_t bar, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          bar),
      "r"(issue)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r));
  return r;
}

__device__ __forceinline__ void tmem_st_16x256b_x8(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x8.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_16x256b_x8(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 16 lanes x 32 columns: thread t receives lanes t / 4 and t / 4 + 8, and of each 8 columns the two
// from 2 (t % 4) on: words 4 j, 4 j + 1 of the first lane, 4 j + 2, 4 j + 3 of the second.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Twice four words of each of four lanes: lane q gets word q of lanes 0 to 3.
__device__ __forceinline__ void quad_transpose(uint32_t (&v)[2][4], uint32_t lane) {
  const bool odd = lane & 1u, upper = lane & 2u;
  uint32_t got[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      got[i][j] = __shfl_xor_sync(0xffffffffu, odd ? v[i][2 * j] : v[i][2 * j + 1], 1);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (odd) v[i][2 * j] = got[i][j];
      else v[i][2 * j + 1] = got[i][j];
    }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      got[i][j] = __shfl_xor_sync(0xffffffffu, upper ? v[i][j] : v[i][j + 2], 2);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (upper) v[i][j] = got[i][j];
      else v[i][j + 2] = got[i][j];
    }
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(addr)
               : "memory");
  return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// x y + z in BF16, two values a word, rounded once.
__device__ __forceinline__ uint32_t bf16x2_fma(uint32_t x, uint32_t y, uint32_t z) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(z));
  return r;
}
__device__ __forceinline__ uint32_t bf16x2_mul(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}
// x y - z.
__device__ __forceinline__ uint32_t bf16x2_residual(uint32_t x, uint32_t y, uint32_t z) {
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\tneg.bf16x2 t, %3;\n\tfma.rn.bf16x2 %0, %1, %2, t;\n\t}"
      : "=r"(r)
      : "r"(x), "r"(y), "r"(z));
  return r;
}
__device__ __forceinline__ uint32_t bf16_twice(float f) { return ptx::pack_bf16x2(f, f); }

// (x0, x1) *= (y0, y1), two FP32 products an instruction.
__device__ __forceinline__ void mul2(uint32_t& x0, uint32_t& x1, float y0, float y1) {
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b64 y, {%2, %3};\n\t"
      "mul.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+r"(x0), "+r"(x1)
      : "f"(y0), "f"(y1));
}

// (x0, x1) += f (y0, y1).
__device__ __forceinline__ void add2(uint32_t& x0, uint32_t& x1, float f, uint32_t y0, uint32_t y1) {
  asm("{\n\t.reg .b64 x, y, f;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b64 y, {%2, %3};\n\t"
      "mov.b64 f, {%4, %4};\n\t"
      "fma.rn.f32x2 x, y, f, x;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+r"(x0), "+r"(x1)
      : "r"(y0), "r"(y1), "f"(f));
}

// Sign bits set where a half word, as BF16, is no finite number.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
__device__ __forceinline__ void st_shared_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// A lane's share of 16 rows x 64 columns of the state in TMEM (the 16x256b layout): rows row and row + 8,
// columns col, col + 1 and those 8, 16, ... further on.  Eight rows' 32-byte sectors an access, where a
// row in each lane would touch 32 rows.
struct StatePart {
  int32_t row, col;
  uint32_t tmem;
};
__device__ __forceinline__ StatePart state_part(uint32_t warp, uint32_t lane, int32_t part) {
  const int32_t half = part & 1, box = part >> 1;
  return {static_cast<int32_t>((warp & 3u) * 32 + 16 * half + lane / 4),
          64 * box + 2 * static_cast<int32_t>(lane & 3u),
          (static_cast<uint32_t>(16 * half) << 16) + 64 * box};
}
__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// e^(g n) from g / ln 2, 1 for n = 0 whatever g.
__device__ __forceinline__ float decay_power(float g2, int32_t n) {
  return n == 0 ? 1.f : exp2f(g2 * static_cast<float>(n));
}

// Byte offset of 16-byte piece `piece` (of 8 channels) of row r in a tile of boxes of `rows` rows.
__device__ __forceinline__ uint32_t tile_offset(uint32_t r, uint32_t piece, uint32_t rows) {
  return (piece >> 3) * rows * 128u + r * 128u + (((piece & 7u) ^ (r & 7u)) << 4);
}

// Tensor maps of A, B and C of every pass.
struct alignas(64) LinearMaps {
  CUtensorMap m[3][3];
};

// A wait of a role whose warps go on together (.sync.aligned accesses to TMEM, votes, __syncwarp): one
// result for all lanes.  Each lane waits for itself, and where some gave up and others did not, those that
// go on would wait in vain for the rest.  (Two votes a wait where the first try fails; the MMA issuer, on
// which the products wait, has no such instructions and goes without.  Level with no votes at all, votes
// there too 0 to 2 %.)
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, const ptx::WaitCtx& ctx,
                                          int32_t site) {
  if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, ptx::mbar_wait_tries(bar, parity, ctx, site));
}

// What a block does: units (a pass's, a sequence's or a segment's tokens of one head) and their chunks.
struct LinearUnit {
  int32_t pass, head;
  bool reverse;
  int64_t first, count;
  int32_t chunks;
  const float* from;  // starting state, null: zeros
  float* to;          // final state, null: not wanted
  float from_factor, to_factor;
  bool transposed;    // from
};

// (Out of line: once per unit in each role.)
template <bool Out>
__device__ __noinline__ LinearUnit linear_unit(const LinearBatch& batch, int32_t each, int32_t u) {
  LinearUnit r = {};
  r.pass = u / each;
  u -= r.pass * each;
  const LinearParams& p = batch.pass[r.pass];
  r.reverse = p.reverse != 0;
  const int32_t at = u / p.heads;
  const int64_t size = static_cast<int64_t>(p.da) * p.dc;
  r.head = u - at * p.heads;
  LinearItem item = {at, 0, 0, 0, 1};
  if (p.items != nullptr) {
    item = p.items[at];
  } else {
    const LinearSpan span = linear_span(p.offsets, at, p.tokens);
    item.first = static_cast<int32_t>(span.first);
    item.count = static_cast<int32_t>(span.count);
  }
  const bool cut = p.segments != nullptr;
  float* const segment = p.segments + (static_cast<int64_t>(at) * p.heads + r.head) * size;
  r.from_factor = r.to_factor = 1.f;
  if constexpr (!Out) {
    if (!item.last)
      r.to = segment + p.heads * size;
    else if (p.final != nullptr)
      r.to = p.segments +
             ((static_cast<int64_t>(p.most_items) + item.sequence) * p.heads + r.head) * size;
    else
      return r;
  } else if (cut) {  // (linear_segments_kernel has written the final state, maybe over the starting one)
    if (item.index > 0 || p.state != nullptr) r.from = segment;
  } else {
    if (p.state != nullptr) {
      const int64_t place = linear_place(p.state_slots, item.sequence, p.state_places);
      if (place >= 0) r.from = p.state + (place * p.heads + r.head) * size;
      r.from_factor = p.state_factor;
      r.transposed = p.state_transposed != 0;
    }
    if (p.final != nullptr) {
      const int64_t place = linear_place(p.final_slots, item.sequence, p.final_places);
      if (place >= 0) r.to = p.final + (place * p.heads + r.head) * size;
      r.to_factor = p.final_factor;
    }
  }
  r.first = item.first;
  r.count = item.count;
  r.chunks = static_cast<int32_t>((r.count + kChunk - 1) / kChunk);
  return r;
}

// The x-th chunk to be done: its first token and how many it has.
__device__ __forceinline__ int32_t chunk_at(const LinearUnit& u, int32_t x, int32_t* count) {
  const int64_t at = static_cast<int64_t>(u.reverse ? u.chunks - 1 - x : x) * kChunk;
  const int64_t left = u.count - at;
  *count = left < kChunk ? static_cast<int32_t>(left) : kChunk;
  return static_cast<int32_t>(u.first + at);
}

// Work::kStates: only the state that each unit leaves, from zeros, and without A.  kFine: see above, kExact:
// outputs with states to FP32 accuracy (variants of their own: decided at run time, they take registers
// that kOutput wants, 2-11 %; the others ask batch.exact).
enum class Work { kStates, kOutput, kFine, kExact };

template <int DA, int DC, Work W>
__global__ void __launch_bounds__(kChunkThreads, 1)
    linear_chunks_kernel(const __grid_constant__ LinearMaps maps,
                         const __grid_constant__ LinearBatch batch) {
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
  using L = ChunkLayout<DA, DC>;
  constexpr bool Out = W != Work::kStates, kFine = W == Work::kFine;
  const bool exact = W == Work::kOutput ? false : W == Work::kExact ? true : batch.exact != 0;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw);
  const uint32_t bars = base + L::kBars;
  // One phase per chunk each; those with two entries, per chunk of the slot.
  const uint32_t a_full = bars, a_empty = bars + 8, b_full = bars + 16, c_full = bars + 32,
                 b_empty = bars + 48, c_empty = bars + 64, s_full = bars + 80, p_ready = bars + 88,
                 o_full = bars + 96, o_free = bars + 104, h_ready = bars + 112,
                 b_ready = bars + 120, h_full = bars + 128, c_ready = bars + 136,
                 drain = bars + 152, small_free = bars + 160;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(base_ptr + L::kSlot);
  volatile int32_t* abort_flag = reinterpret_cast<volatile int32_t*>(base_ptr + L::kSlot + 4);
  const uint32_t warp = threadIdx.x >> 5;
  const uint32_t lane = ptx::lane_id();

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < L::kNumBars; ++i) {
      const uint32_t bar = bars + 8 * i;
      ptx::mbar_init(bar, bar == o_free ? 8
                          : bar == p_ready || bar == h_ready || bar == b_ready || bar == small_free ? 4
                          : bar == c_ready || bar == c_ready + 8 ? 2
                                                                 : 1);
    }
    *abort_flag = 0;
    ptx::fence_mbarrier_init_cluster();
    ptx::fence_proxy_async_shared();
  }
  if (warp == 0 && lane < 3 && batch.pass[0].tokens > 0) ptx::prefetch_tensormap(&maps.m[0][lane]);
  if (warp == 1) {
    ptx::tmem_alloc<1>(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    ptx::tmem_relinquish<1>();
  }
  uint32_t* bad = reinterpret_cast<uint32_t*>(base_ptr + L::kBad);
  volatile uint32_t* last_bad = bad + kChunk;
  // Chunks that each warp of the output has done, and that each of the state has begun.
  volatile uint32_t* done = bad + kChunk + 4;
  if (threadIdx.x < kChunk + 16) bad[threadIdx.x] = 0u;
  kernel_begins();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const ptx::WaitCtx ctx{abort_flag, &linear_status_word, batch.timeout_ns};
  const LinearParams& any = batch.pass[0];
  const int32_t each = (any.items != nullptr ? *any.item_count : any.sequences) * any.heads;
  const int32_t units = each * batch.passes;
  // Units in rounds of one per block, to and fro: in order of their lengths, that evens out the blocks.
  auto unit_at = [](int32_t round) {
    const int32_t step = static_cast<int32_t>(gridDim.x), b = static_cast<int32_t>(blockIdx.x);
    return round * step + (round & 1 ? step - 1 - b : b);
  };
  // Thread of a warpgroup: the token of the chunk, or the row of the state, that it has, and the TMEM
  // lanes of its warp.
  const int32_t i = static_cast<int32_t>(threadIdx.x & 127u);
  const uint32_t lanes = tmem + ((warp & 3u) << 21);
  uint32_t n = 0;  // chunks done
  bool ok = true;
  // C's slot of chunk m and the parity of its phases.
  const bool one_c = L::kShared && exact;
  auto c_slot = [&](uint32_t m) { return one_c ? 0u : m & 1u; };
  auto c_phase = [&](uint32_t m) { return one_c ? m & 1u : (m >> 1) & 1u; };

  if (warp == 0) {
    // ---------------------------------------------------------------------------- producer
    if (lane == 0) {
      const uint64_t policy = ptx::policy_evict_first();
      const bool skip_all = batch.inject & kLinearSkipLoads;
      const bool skip_c = batch.inject & (kLinearSkipLoads | kLinearSkipValues);
      uint32_t end_a = 0, end_b = 0, end_c = 0;  // one past the last chunk whose tile is on its way
      for (int32_t r = 0, u = unit_at(0); u < units && ok; u = unit_at(++r)) {
        const LinearUnit unit = linear_unit<Out>(batch, each, u);
        const LinearParams& p = batch.pass[unit.pass];
        const CUtensorMap *tm_a = &maps.m[unit.pass][0], *tm_b = &maps.m[unit.pass][1],
                          *tm_c = &maps.m[unit.pass][2];
        const int32_t ha = unit.head / p.a.share, hb = unit.head / p.b.share,
                      hc = unit.head / p.c.share;
#pragma unroll 1
        for (int32_t x = 0; x < unit.chunks; ++x, ++n) {
          int32_t count;
          const int32_t t = chunk_at(unit, x, &count);
          const uint32_t slot = n & 1u;
          const uint32_t b = base + L::kB + slot * L::kTileA;
          const uint32_t c = base + L::kC + c_slot(n) * L::kTileC;
          const uint32_t cf = c_full + 8 * c_slot(n);
          if (!(ok = ptx::mbar_wait_brief(b_empty + 8 * slot, ((n >> 1) & 1u) ^ 1u, ctx,
                                          kSiteLinearProducer)))
            break;
          if (skip_all) continue;
          ptx::mbar_arrive_expect_tx(b_full + 8 * slot, L::kTileA);
          for (int j = 0; j < DA / 64; ++j)
            ptx::tma_load_3d(tm_b, b + j * 16384, b_full + 8 * slot, 64 * j, hb, t, policy);
          end_b = n + 1;
          // What waits for room below comes into L2 meanwhile.
          if (Out)
            for (int j = 0; j < DA / 64; ++j) ptx::tma_prefetch_l2_3d(tm_a, 64 * j, ha, t);
          if (one_c)
            for (int j = 0; j < DC / 64; ++j) ptx::tma_prefetch_l2_3d(tm_c, 64 * j, hc, t);
          // C first unless its only slot is the last to become free.
          for (int turn = 0; turn < 2 && ok; ++turn) {
            if ((turn == 0) == one_c) {
              if (!Out) continue;
              if (!(ok = ptx::mbar_wait_brief(a_empty, (n & 1u) ^ 1u, ctx, kSiteLinearProducer)))
                break;
              ptx::mbar_arrive_expect_tx(a_full, L::kTileA);
              for (int j = 0; j < DA / 64; ++j)
                ptx::tma_load_3d(tm_a, base + L::kA + j * 16384, a_full, 64 * j, ha, t, policy);
              end_a = n + 1;
            } else {
              if (!(ok = ptx::mbar_wait_brief(c_empty + 8 * c_slot(n), c_phase(n) ^ 1u, ctx,
                                              kSiteLinearProducer)))
                break;
              if (skip_c) continue;
              ptx::mbar_arrive_expect_tx(cf, L::kTileC);
              for (int j = 0; j < DC / 64; ++j)
                ptx::tma_load_3d(tm_c, c + j * 16384, cf, 64 * j, hc, t, policy);
              end_c = n + 1;
            }
          }
          if (!ok) break;
        }
      }
      // The copies land before the block ends, whichever role has given up: the last in every slot, as a
      // slot is filled again only after the copy before has.
      volatile int32_t none = 0;
      const ptx::WaitCtx brief{&none, nullptr, kLinearDrainNs};
      auto landed = [&](uint32_t bar, uint32_t parity) {
        none = 0;
        ptx::mbar_wait_brief(bar, parity, brief, kSiteLinearDrain);
      };
#pragma unroll 1
      for (uint32_t j = end_b > 2 ? end_b - 2 : 0; j < end_b; ++j)
        landed(b_full + 8 * (j & 1u), (j >> 1) & 1u);
      const uint32_t slots_c = one_c ? 1 : 2;
#pragma unroll 1
      for (uint32_t j = end_c > slots_c ? end_c - slots_c : 0; j < end_c; ++j)
        landed(c_full + 8 * c_slot(j), c_phase(j));
      if (end_a > 0) landed(a_full, (end_a - 1) & 1u);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------------------- MMA issuer
    {
      // (Each lane waits, and may give up, for itself: the issuing lane alone makes products, and the others
      // do not take part in anything before the end.)
      const uint32_t issue = elect_one();
      constexpr uint32_t kScores = linear_idesc(kChunk, false, false);
      constexpr uint32_t kInter = linear_idesc(DC, false, true);
      constexpr uint32_t kState = linear_idesc(DC, true, true);
      const uint32_t a_k = ptx::sw128_desc_lo(base + L::kA);  // A along its channels
      const uint32_t s_mn = desc_lo_mn(base + L::kS, DA * 128);
      for (int32_t r = 0, u = unit_at(0); u < units && ok; u = unit_at(++r)) {
        const LinearUnit unit = linear_unit<Out>(batch, each, u);
        bool state = unit.from != nullptr;
#pragma unroll 1
        for (int32_t x = 0; x < unit.chunks && ok; ++x, ++n) {
          int32_t count;
          chunk_at(unit, x, &count);
          const uint32_t slot = n & 1u, twice = (n >> 1) & 1u, once = n & 1u;
          const uint32_t b = base + L::kB + slot * L::kTileA;
          const uint32_t c_mn = desc_lo_mn(base + L::kC + c_slot(n) * L::kTileC, 16384);
          if constexpr (Out) {
            // A B^T.  Its columns hold P of the chunk before until that one's product is done, and then
            // the small parts of the state's addend until they have been added.
            if (n > 0) ok = ptx::mbar_wait_brief(o_full, once ^ 1u, ctx, kSiteLinearMma);
            if (n > 0 && exact)
              ok = ok && ptx::mbar_wait_brief(small_free, once ^ 1u, ctx, kSiteLinearMma);
            ok = ok && ptx::mbar_wait_brief(a_full, once, ctx, kSiteLinearMma) &&
                 ptx::mbar_wait_brief(b_full + 8 * slot, twice, ctx, kSiteLinearMma);
            if (!ok) break;
            ptx::tc_fence_after();
            const uint32_t b_k = ptx::sw128_desc_lo(b);
#pragma unroll
            for (int k = 0; k < DA / 16; ++k)
              umma_f16_ss(tmem + kColScores, a_k + k_step(k), b_k + k_step(k), kScores, k > 0, issue);
            umma_commit_if(s_full, issue);
            // A S into its own columns, once the output before has been read.
            ok = ptx::mbar_wait_brief(h_ready, once, ctx, kSiteLinearMma);
            if (n > 0) ok = ok && ptx::mbar_wait_brief(o_free, once ^ 1u, ctx, kSiteLinearMma);
            if (!ok) break;
            ptx::tc_fence_after();
            if (state) {
#pragma unroll
              for (int k = 0; k < DA / 16; ++k)
                umma_f16_ss(tmem + kColInter, a_k + k_step(k), s_mn + k * 128, kInter, k > 0, issue);
            }
            umma_commit_if(a_empty, issue);
            // P C.  A partial chunk's rows of C past its end are cleared before b_ready.
            ok = ptx::mbar_wait_brief(p_ready, once, ctx, kSiteLinearMma) &&
                 ptx::mbar_wait_brief(c_full + 8 * c_slot(n), c_phase(n), ctx, kSiteLinearMma) &&
                 ptx::mbar_wait_brief(c_ready + 8 * slot, twice, ctx, kSiteLinearMma) &&
                 (count == kChunk || ptx::mbar_wait_brief(b_ready, once, ctx, kSiteLinearMma));
            if (!ok) break;
            ptx::tc_fence_after();
            if constexpr (!kFine) {
#pragma unroll
              for (int k = 0; k < kChunk / 16; ++k)
                umma_f16_ts(tmem + kColIntra, tmem + kColScores + k * 8, c_mn + k * 128, kInter, k > 0,
                            issue);
            } else {
#pragma unroll 1
              for (int k = 0; k < kChunk / 8; ++k)  // both parts of 16 tokens
                umma_f16_ts(tmem + kColIntra, tmem + kColScores + 32 * (k >> 2) + 8 * (k & 3),
                            c_mn + ((k >> 2) * 2 + (k & 1)) * 128, kInter, k > 0, issue);
            }
            umma_commit_if(o_full, issue);
          } else {
            ok = ptx::mbar_wait_brief(h_ready, once, ctx, kSiteLinearMma) &&
                 ptx::mbar_wait_brief(c_full + 8 * c_slot(n), c_phase(n), ctx, kSiteLinearMma) &&
                 ptx::mbar_wait_brief(c_ready + 8 * slot, twice, ctx, kSiteLinearMma);
            if (!ok) break;
          }
          // The state's addend, by the parts of left . B.
          if (!(ok = ptx::mbar_wait_brief(b_ready, once, ctx, kSiteLinearMma))) break;
          ptx::tc_fence_after();
          uint32_t accumulate = state ? 1u : 0u, sum = kColState;
#pragma unroll 1
          for (int j = 0; j < (exact ? 3 : 2); ++j) {
            if (exact && j == 1) {  // over P
              if (Out && !(ok = ptx::mbar_wait_brief(o_full, once, ctx, kSiteLinearMma))) break;
              ptx::tc_fence_after();
              accumulate = 0u;
              sum = kColScores;
            }
            const uint32_t part =
                desc_lo_mn(j == 0 ? b : base + (j == 1 ? L::kMid : L::kLo), 16384);
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k) {
              umma_f16_ss(tmem + sum, part + k * 128, c_mn + k * 128, kState, accumulate, issue);
              accumulate = 1u;
            }
          }
          if (!ok) break;
          umma_commit_if(b_empty + 8 * slot, issue);
          umma_commit_if(c_empty + 8 * c_slot(n), issue);
          umma_commit_if(h_full, issue);
          state = true;
        }
      }
      // The products end before TMEM is freed, whichever role has given up.
      volatile int32_t none = 0;
      umma_commit_if(drain, issue);
      ptx::mbar_wait_brief(drain, 0, {&none, nullptr, kLinearDrainNs}, kSiteLinearDrain);
    }
    __syncwarp();
  } else if (warp < 4) {
    // ----------------------------------------------------------- infinities and NaN in a box of C
    const uint32_t box = warp - 2;
    for (int32_t r = 0, u = unit_at(0); u < units && ok; u = unit_at(++r)) {
      const LinearUnit unit = linear_unit<Out>(batch, each, u);
      const bool reverse = unit.reverse;
      const uint32_t unit_first = n * kChunk;  // place of the unit's first token in the block's work
#pragma unroll 1
      for (int32_t x = 0; x < unit.chunks; ++x, ++n) {
        int32_t count;
        chunk_at(unit, x, &count);
        const uint32_t c = base + L::kC + c_slot(n) * L::kTileC + box * 16384;
        if (!(ok = wait_warp(c_full + 8 * c_slot(n), c_phase(n), ctx, kSiteLinearScan)))
          break;
        uint32_t found = 0;
        if (box < DC / 64) {
#pragma unroll 1
          for (int32_t row = static_cast<int32_t>(lane); row < count; row += 32)
#pragma unroll
            for (uint32_t piece = 0; piece < 8; ++piece) {
              const uint4 v = ld_shared_v4(c + tile_offset(row, piece, kChunk));
              found |= not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w);
            }
        }
        if (__any_sync(0xffffffffu, found != 0u)) {
          // The table is the earlier chunks' outputs' and the unit before's state's until then.
          const uint64_t t0 = ptx::globaltimer();
          while (ok && !__all_sync(0xffffffffu, lane >= 12 || (lane < 8 && !Out) ||
                                              done[lane] >= n + (lane < 8 ? 0u : 1u))) {
            const bool late = ptx::globaltimer() - t0 > ctx.timeout_ns;
            if (late) ptx::record_timeout(ctx, kSiteLinearScan);
            ok = !__any_sync(0xffffffffu, late || *abort_flag != 0);
          }
          if (!ok) break;
          uint32_t* mine = bad + 64 * box + 2 * lane;  // of the two channels a lane has
#pragma unroll 1
          for (int32_t place = reverse ? kChunk - count : 0; place < (reverse ? kChunk : count);
               ++place) {
            const int32_t row = reverse ? kChunk - 1 - place : place;
            const uint32_t at = c + tile_offset(row, lane / 4, kChunk) + 4 * (lane & 3u);
            const uint32_t v = ptx::ld_shared_u32(at), f = not_finite(v);
            if (f == 0) continue;
            st_shared_u32(at, v & ((f & 0x8000u ? 0u : 0xffffu) | (f >> 16 ? 0u : 0xffff0000u)));
            const uint32_t here = n * kChunk + place + 1;
            if ((f & 0x8000u) && mine[0] <= unit_first) mine[0] = here;
            if ((f >> 16) && mine[1] <= unit_first) mine[1] = here;
          }
          __syncwarp();
          if (lane == 0) *last_bad = n * kChunk + kChunk;
          ptx::fence_proxy_async_shared();
          __syncwarp();
        }
        if (lane == 0) ptx::mbar_arrive(c_ready + 8 * (n & 1u));
      }
    }
  } else if (Out && warp >= 4 && warp < 8) {
    // ------------------------------------------------------------------------- scores -> P
    const uint32_t w = warp - 4;
    // scale e^(g |m - 32|): with 32 + (this token) - (another of its 32) for m the decay between them, and
    // with the other's place for m the decay to 32 others but for a factor of the block (each
    // factor an exponent of one sign, so that none is above 1).
    float* powers = reinterpret_cast<float*>(base_ptr + L::kPowers) + 64 * w;
    const float* own = powers + 32 + lane;
    for (int32_t r = 0, u = unit_at(0); u < units && ok; u = unit_at(++r)) {
      const LinearUnit unit = linear_unit<Out>(batch, each, u);
      const LinearParams& p = batch.pass[unit.pass];
      const bool reverse = unit.reverse;
      const float g2 = p.log_decay[unit.head] * 1.4426950408889634f;
      const float* others = powers + (reverse ? 32 : 0);
      // Which of the warp's tokens each sees.
      const uint32_t seen = reverse ? 0xffffffffu << lane : 0xffffffffu >> (31u - lane);
      __syncwarp();
      powers[lane] = p.scale * decay_power(g2, 32 - static_cast<int32_t>(lane));
      powers[lane + 32] = p.scale * decay_power(g2, static_cast<int32_t>(lane));
      __syncwarp();
#pragma unroll 1
      for (int32_t x = 0; x < unit.chunks; ++x, ++n) {
        int32_t count;
        chunk_at(unit, x, &count);
        if (!(ok = wait_warp(s_full, n & 1u, ctx, kSiteLinearScores))) break;
        ptx::tc_fence_after();
#pragma unroll 1
        for (uint32_t blk = 0; blk < 4; ++blk) {
          uint32_t s[32];
          if (reverse ? blk < w : blk > w) {
#pragma unroll
            for (int k = 0; k < 16; ++k) s[k] = 0u;
          } else {
            ptx::tmem_ld_32x32b_x32(lanes + kColScores + 32 * blk, s);
            ptx::tmem_ld_wait();
            if (blk == w) {
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                const float f = __uint_as_float(s[k]) * own[-k];
                s[k] = seen & (1u << k) ? __float_as_uint(f) : 0u;
              }
            } else {
              const int32_t first = static_cast<int32_t>(32 * blk);
              const float r = decay_power(g2, reverse ? first - i : i - first - 32);
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                const float4 d = *reinterpret_cast<const float4*>(others + k);
                mul2(s[k], s[k + 1], r, r);
                mul2(s[k + 2], s[k + 3], r, r);
                mul2(s[k], s[k + 1], d.x, d.y);
                mul2(s[k + 2], s[k + 3], d.z, d.w);
              }
            }
            // (In order, tokens past the end are later than any whose output is kept.)
            if (reverse && count < kChunk) {
              const int32_t left = count - static_cast<int32_t>(32 * blk);
#pragma unroll
              for (int k = 0; k < 32; ++k) s[k] = k < left ? s[k] : 0u;
            }
            if constexpr (kFine) {  // the second part, over the second half of this block's scores
              uint32_t low[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const float x = __uint_as_float(s[2 * k]), y = __uint_as_float(s[2 * k + 1]);
                s[k] = ptx::pack_bf16x2(x, y);
                low[k] = ptx::pack_bf16x2(x - bf16_lo(s[k]), y - bf16_hi(s[k]));
              }
              tmem_st_32x32b_x16(lanes + kColScores + 32 * blk + 16, low);
            } else {
#pragma unroll
              for (int k = 0; k < 16; ++k)
                s[k] = ptx::pack_bf16x2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1]));
            }
          }
          // Over scores that this lane has read: those of blocks up to this one.
          const uint32_t packed[16] = {s[0], s[1], s[2],  s[3],  s[4],  s[5],  s[6],  s[7],
                                       s[8], s[9], s[10], s[11], s[12], s[13], s[14], s[15]};
          tmem_st_32x32b_x16(lanes + kColScores + (kFine ? 32 : 16) * blk, packed);
          if (kFine && (reverse ? blk < w : blk > w))
            tmem_st_32x32b_x16(lanes + kColScores + 32 * blk + 16, packed);  // zeros too
        }
        tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_ready);
      }
    }
  } else if (Out && warp >= 8 && warp < 16) {
    // ------------------------------------------------------------------------------ output
    constexpr int kCols = DC / 2;  // of each of the two warps that share TMEM lanes
    const int32_t col0 = static_cast<int32_t>((warp - 8) / 4) * kCols;
    for (int32_t r = 0, u = unit_at(0); u < units && ok; u = unit_at(++r)) {
      const LinearUnit unit = linear_unit<Out>(batch, each, u);
      const LinearParams& p = batch.pass[unit.pass];
      const bool reverse = unit.reverse;
      const float g2 = p.log_decay[unit.head] * 1.4426950408889634f;
      const uint32_t unit_first = n * kChunk;
      bool state = unit.from != nullptr;
#pragma unroll 1
      for (int32_t x = 0; x < unit.chunks; ++x, ++n) {
        int32_t count;
        const int64_t t = chunk_at(unit, x, &count);
        if (!(ok = wait_warp(o_full, n & 1u, ctx, kSiteLinearOutput))) break;
        ptx::tc_fence_after();
        const bool spoilt = *last_bad > unit_first;
        // 16 tokens x 32 channels at a time: a lane has neighbouring pairs of channels of two tokens,
        // four lanes a token's eight channels.  (A token's channels in one lane would make each
        // store touch 32 rows: 2270 cycles of the SM's data path a chunk, which the products need.)
#pragma unroll 1
        for (int32_t half = 0; half < 2; ++half) {
          const int32_t token = static_cast<int32_t>((warp & 3u) * 32 + 16 * half + lane / 4);
          float since[2];
          int64_t row[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int32_t at = token + 8 * r;
            since[r] = p.scale * decay_power(g2, reverse ? max(count - 1 - at, 0) : at + 1);
            row[r] = (t + at) * p.o_token + unit.head * p.o_head;
          }
#pragma unroll 1
          for (int32_t col = col0; col < col0 + kCols; col += 32) {
            const uint32_t at = lanes + (static_cast<uint32_t>(16 * half) << 16) + col;
            uint32_t o[16], s[16];
            __syncwarp();
            tmem_ld_16x256b_x4(at + kColIntra, o);
            if (state) tmem_ld_16x256b_x4(at + kColInter, s);
            ptx::tmem_ld_wait();
            if (state) {
#pragma unroll
              for (int j = 0; j < 16; j += 2)
                add2(o[j], o[j + 1], since[(j >> 1) & 1], s[j], s[j + 1]);
            }
            if (spoilt) {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const int32_t at = token + 8 * ((j >> 1) & 1);
                const uint32_t first =
                    bad[col + 8 * (j / 4) + 2 * static_cast<int32_t>(lane & 3u) + (j & 1)];
                const uint32_t here = n * kChunk + (reverse ? kChunk - 1 - at : at) + 1;
                if (first > unit_first && here >= first) o[j] = 0x7fc00000u;
              }
            }
            if (p.o_f32) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int32_t channel = col + 8 * (j / 2) + 2 * static_cast<int32_t>(lane & 3u);
                if (token + 8 * (j & 1) < count && channel < p.dc)
                  *reinterpret_cast<uint2*>(static_cast<float*>(p.o) + row[j & 1] + channel) =
                      make_uint2(o[2 * j], o[2 * j + 1]);
              }
              continue;
            }
            uint32_t v[2][4];  // of both tokens
#pragma unroll
            for (int j = 0; j < 8; ++j)
              v[j & 1][j / 2] =
                  ptx::pack_bf16x2(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]));
            quad_transpose(v, lane);
            const int32_t channel = col + 8 * static_cast<int32_t>(lane & 3u);
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (token + 8 * j < count && channel < p.dc)
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.o) + row[j] + channel) =
                    make_uint4(v[j][0], v[j][1], v[j][2], v[j][3]);
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(o_free);
          done[warp - 8] = n + 1;
        }
        state = true;
      }
    }
  } else if (warp >= 16 && warp < 20) {
    // --------------------------------------------------------------------------- the state
    const uint32_t mine = lanes + kColState;
    for (int32_t r = 0, u = unit_at(0); u < units && ok; u = unit_at(++r)) {
      const LinearUnit unit = linear_unit<Out>(batch, each, u);
      const LinearParams& p = batch.pass[unit.pass];
      const float g2 = p.log_decay[unit.head] * 1.4426950408889634f;
      const uint32_t unit_first = n * kChunk;
      const float* from = unit.from;
      float* to = unit.to;
      auto starting = [&](int32_t c) {  // column c of row i of the starting state
        return from != nullptr && i < p.da && c < p.dc
                   ? unit.from_factor * from[unit.transposed ? c * p.da + i : i * p.dc + c]
                   : 0.f;
      };
      if (unit.chunks == 0) {  // the final state is the starting one (no pass has both one and a transposed one)
        const float factor = unit.from_factor * unit.to_factor;
        const int32_t size = p.da * p.dc;
        if (to == nullptr || (to == from && factor == 1.f)) continue;
        for (int32_t e0 = 4 * i; e0 < size; e0 += 4 * 128 * 4) {  // four loads in flight
          float4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int32_t e = e0 + 4 * 128 * k;
            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (from != nullptr && e < size) v[k] = *reinterpret_cast<const float4*>(from + e);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (e0 + 4 * 128 * k < size)
              *reinterpret_cast<float4*>(to + e0 + 4 * 128 * k) =
                  make_float4(factor * v[k].x, factor * v[k].y, factor * v[k].z, factor * v[k].w);
        }
        continue;
      }
      if (from != nullptr && unit.transposed) {
#pragma unroll 1
        for (int32_t col = 0; col < DC; col += 16) {
          uint32_t s[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) s[k] = __float_as_uint(starting(col + k));
          __syncwarp();
          tmem_st_32x32b_x16(mine + col, s);
        }
        tmem_st_wait();
      } else if (from != nullptr) {
#pragma unroll 1
        for (int32_t part = 0; part < DC / 32; ++part) {
          const StatePart at = state_part(warp, lane, part);
          const float* tile = from + at.row * p.dc + at.col;
          uint32_t s[32];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float2 v = make_float2(0.f, 0.f);
            if (at.row + 8 * (k & 1) < p.da && at.col + 8 * (k / 2) < p.dc)
              v = *reinterpret_cast<const float2*>(tile + 8 * (k & 1) * p.dc + 8 * (k / 2));
            s[2 * k] = __float_as_uint(unit.from_factor * v.x);
            s[2 * k + 1] = __float_as_uint(unit.from_factor * v.y);
          }
          __syncwarp();
          tmem_st_16x256b_x8(mine + at.tmem, s);
        }
        tmem_st_wait();
      }
      // The next unit's on its way from memory meanwhile.
      if (const int32_t next = unit_at(r + 1); Out && next < units) {
        const LinearUnit later = linear_unit<Out>(batch, each, next);
        if (later.from != nullptr)
          for (int32_t line = i; line < p.da * p.dc / 32; line += 128)
            prefetch_l2(later.from + 32 * line);
      }
#pragma unroll 1
      for (int32_t x = 0; x < unit.chunks; ++x, ++n) {
        int32_t count;
        chunk_at(unit, x, &count);
        const float decay = decay_power(g2, count);
        // The chunk before is done with the state and its copy (at a unit's first chunk: waited for
        // at the end of the last one).
        if (x > 0) {
          if (!(ok = wait_warp(h_full, (n - 1) & 1u, ctx, kSiteLinearState))) break;
          ptx::tc_fence_after();
        }
        if ((warp & 3u) * 32 < DA && (x > 0 || from != nullptr)) {
#pragma unroll 1
          for (int32_t col = 0; col < DC; col += 16) {
            uint32_t s[16];
            ptx::tmem_ld_32x32b_x16(mine + col, s);
            if (exact && x > 0) {
              uint32_t small[16];
              ptx::tmem_ld_32x32b_x16(lanes + kColScores + col, small);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; k += 2) add2(s[k], s[k + 1], 1.f, small[k], small[k + 1]);
            }
            ptx::tmem_ld_wait();
            if constexpr (Out) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              ptx::st_shared_v4(
                  base + L::kS + tile_offset(i, col / 8 + k, DA),
                  ptx::pack_bf16x2(__uint_as_float(s[8 * k]), __uint_as_float(s[8 * k + 1])),
                  ptx::pack_bf16x2(__uint_as_float(s[8 * k + 2]), __uint_as_float(s[8 * k + 3])),
                  ptx::pack_bf16x2(__uint_as_float(s[8 * k + 4]), __uint_as_float(s[8 * k + 5])),
                  ptx::pack_bf16x2(__uint_as_float(s[8 * k + 6]), __uint_as_float(s[8 * k + 7])));
            }
#pragma unroll
            for (int k = 0; k < 16; k += 2) mul2(s[k], s[k + 1], decay, decay);
            tmem_st_32x32b_x16(mine + col, s);
          }
          tmem_st_wait();
        }
        ptx::fence_proxy_async_shared();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(h_ready);
          if (exact && x > 0) ptx::mbar_arrive(small_free);
          done[warp - 8] = n + 1;
        }
      }
      if (!ok || !(ok = wait_warp(h_full, (n - 1) & 1u, ctx, kSiteLinearState))) break;
      ptx::tc_fence_after();
      if (to != nullptr) {
        const bool spoilt = *last_bad > unit_first;
#pragma unroll 1
        for (int32_t part = 0; part < DC / 16; ++part) {  // half a part: 32 columns
          StatePart at = state_part(warp, lane, part / 2);
          at.col += 32 * (part & 1);
          at.tmem += 32 * (part & 1);
          float* tile = to + at.row * p.dc + at.col;
          uint32_t s[16];
          __syncwarp();
          tmem_ld_16x256b_x4(mine + at.tmem, s);
          if (exact) {
            uint32_t small[16];
            tmem_ld_16x256b_x4(lanes + kColScores + at.tmem, small);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; k += 2) add2(s[k], s[k + 1], 1.f, small[k], small[k + 1]);
          }
          ptx::tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int32_t col = at.col + 8 * (k / 2);
            float2 v = make_float2(unit.to_factor * __uint_as_float(s[2 * k]),
                                   unit.to_factor * __uint_as_float(s[2 * k + 1]));
            if (spoilt) {
              if (bad[col] > unit_first) v.x = __uint_as_float(0x7fc00000u);
              if (bad[col + 1] > unit_first) v.y = __uint_as_float(0x7fc00000u);
            }
            if (at.row + 8 * (k & 1) < p.da && col < p.dc)
              *reinterpret_cast<float2*>(tile + 8 * (k & 1) * p.dc + 8 * (k / 2)) = v;
          }
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0 && exact) ptx::mbar_arrive(small_free);
    }
  } else if (warp >= 20) {
    // ----------------------------------------------------------------------------- left . B
    for (int32_t r = 0, u = unit_at(0); u < units && ok; u = unit_at(++r)) {
      const LinearUnit unit = linear_unit<Out>(batch, each, u);
      const LinearParams& p = batch.pass[unit.pass];
      const bool reverse = unit.reverse;
      const float g2 = p.log_decay[unit.head] * 1.4426950408889634f;
#pragma unroll 1
      for (int32_t x = 0; x < unit.chunks; ++x, ++n) {
        int32_t count;
        chunk_at(unit, x, &count);
        const uint32_t slot = n & 1u, twice = (n >> 1) & 1u;
        const uint32_t b = base + L::kB + slot * L::kTileA;
        const bool inside = i < count;
        const float left = inside ? decay_power(g2, reverse ? i + 1 : count - 1 - i) : 0.f;
        // In place of B, once the scores are made; the second part's tile is the chunk
        // before's until its product is done.
        ok = ptx::mbar_wait_brief(b_full + 8 * slot, twice, ctx, kSiteLinearLeft) &&
             (!Out || ptx::mbar_wait_brief(s_full, n & 1u, ctx, kSiteLinearLeft));
        if (ok && n > 0) ok = ptx::mbar_wait_brief(h_full, (n - 1) & 1u, ctx, kSiteLinearLeft);
        if (ok && count < kChunk)
          ok = ptx::mbar_wait_brief(c_full + 8 * c_slot(n), c_phase(n), ctx, kSiteLinearLeft);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;  // (together, as wait_warp)
        if (exact) {
#pragma unroll 1
          for (uint32_t piece = 0; piece < DA / 8; ++piece) {
            const uint32_t at = tile_offset(i, piece, kChunk);
            const uint4 v = ld_shared_v4(b + at);
            const uint32_t word[4] = {v.x, v.y, v.z, v.w};
            uint32_t hi[4], mid[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float f0 = inside ? bf16_lo(word[k]) * left : 0.f;
              const float f1 = inside ? bf16_hi(word[k]) * left : 0.f;
              hi[k] = ptx::pack_bf16x2(f0, f1);
              const float m0 = f0 - bf16_lo(hi[k]), m1 = f1 - bf16_hi(hi[k]);
              mid[k] = ptx::pack_bf16x2(m0, m1);
              lo[k] = ptx::pack_bf16x2(m0 - bf16_lo(mid[k]), m1 - bf16_hi(mid[k]));
            }
            ptx::st_shared_v4(b + at, hi[0], hi[1], hi[2], hi[3]);
            ptx::st_shared_v4(base + L::kMid + at, mid[0], mid[1], mid[2], mid[3]);
            ptx::st_shared_v4(base + L::kLo + at, lo[0], lo[1], lo[2], lo[3]);
          }
        } else {
          // With left = l1 + l2 to 2^-17 (BF16 parts) and y an element of B: the first part is
          // h = RN(y l1), and y l1 - h, which BF16 holds, + y l2 rounded is the second.
          const uint32_t l1 = bf16_twice(left);
          const uint32_t l2 = bf16_twice(left - bf16_lo(l1));
          const uint32_t mine = static_cast<uint32_t>(i) * 128u + ((static_cast<uint32_t>(i) & 7u) << 4);
#pragma unroll 1
          for (uint32_t half = 0; half < DA / 32; ++half) {  // 32 channels (where tile_offset has them)
            const uint32_t from = (b + (half / 2) * 16384 + mine) ^ ((half & 1u) << 6);
            const uint32_t to = (base + L::kMid + (half / 2) * 16384 + mine) ^ ((half & 1u) << 6);
            uint32_t word[16];
#pragma unroll
            for (uint32_t piece = 0; piece < 4; ++piece) {
              const uint4 v = ld_shared_v4(from ^ (piece << 4));
              word[4 * piece] = v.x;
              word[4 * piece + 1] = v.y;
              word[4 * piece + 2] = v.z;
              word[4 * piece + 3] = v.w;
            }
#pragma unroll
            for (uint32_t piece = 0; piece < 4; ++piece) {
              uint32_t hi[4], mid[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t y = inside ? word[4 * piece + k] : 0u;
                hi[k] = bf16x2_mul(y, l1);
                mid[k] = bf16x2_fma(y, l2, bf16x2_residual(y, l1, hi[k]));
              }
              ptx::st_shared_v4(from ^ (piece << 4), hi[0], hi[1], hi[2], hi[3]);
              ptx::st_shared_v4(to ^ (piece << 4), mid[0], mid[1], mid[2], mid[3]);
            }
          }
        }
        if (!inside) {  // other sequences' rows, or none
          const uint32_t c = base + L::kC + c_slot(n) * L::kTileC;
#pragma unroll 1
          for (uint32_t piece = 0; piece < DC / 8; ++piece)
            ptx::st_shared_v4(c + tile_offset(i, piece, kChunk), 0u, 0u, 0u, 0u);
        }
        ptx::fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(b_ready);
      }
    }
  }
  // Every copy has landed and every product has completed (waited for by the roles that began them).
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc<1>(tmem, 512);
#endif
}

}  // namespace cpg
