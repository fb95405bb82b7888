// Chunk attention on the 5th-generation tensor cores: fp16, bf16 and 8-bit caches, head_dim up to 256, pages of a multiple of
// 8 tokens, groups of up to 128 query heads.
//
// Rows are the (token, query head) pairs of one KV head, 128 a tile (128 / group tokens), two tiles a block (one for head_dim above 128). A
// unit of work is a block and 128 of its keys:
//   S_t = Q_t K^T (M = 128 rows, N = 128 keys) into tensor memory, by one thread, for the tiles t = 0, 1;
//   a warpgroup a tile, one thread a row: the row's maximum, P_t = exp2(S_t - max) back into tensor memory over
//   S_t, in 16 bits; O_t is rescaled in place only when a row's maximum has grown by more than 2^8;
//   O_t += P_t V (A from tensor memory, V as an MN-major operand), by the same thread.
// The two tiles alternate: one's softmax runs under the other's products, which complete in the order of issue, so
// that S_t of the next unit says that O_t += P_t V of this one is done.
// K and V tiles come by TMA through a ring of 128-key stages: a box per page (or 128 keys of it), zeros past the
// sequence's end and for pages outside the pool.
//
// Units are numbered over sequences, KV heads, blocks and keys; every CTA takes an equal run of them, so causal
// triangles, ragged lengths and few rows over long contexts are all balanced the same way. A block that the runs
// cut leaves pieces (O in fp32, maximum, sum) in scratch; of each 32 rows the warp that arrives last joins them in
// the pieces' order.
//
// What is masked does not count whatever it holds: scores are replaced, not added to; a warp clears the V rows
// past the sequence's end and looks for infinities and NaN in rows that some row of the block does not see, in which
// case the softmax threads add that unit's P V themselves, key by key.
//
// Bound by the chain S -> softmax -> P -> products of a tile: 3,700 cycles a unit for its two tiles, of which the products
// take 2,048. A prompt of 8192 tokens with 32/8 heads of 128, bf16, called over and over on changing inputs: 629 us,
// 874 TFLOP/s, 0.52 of the measured matrix product (under the power cap; in runs of 20 calls 571 us). 8 x 512 tokens over
// up to 8192 of 64/8 heads in e4m3 blocks: 1,195 us, 643 TFLOP/s in bf16, 1,205 us in fp16.
#include <cuda.h>

#include <algorithm>
#include <climits>
#include <mutex>
#include <type_traits>

#include "chunk_attention.cuh"

namespace klb {
namespace chunk_attention {

namespace tc {  // named: an unnamed one's name, and with it the register allocation, would follow the comments

constexpr int kBN = 128;                 // keys of a unit
constexpr int kLoadWarp = 8, kMmaWarp = 9, kFixWarp = 11, kWidenWarp = 12;
constexpr float kLazy = 8.0f;            // log2 by which a maximum may be passed before O is rescaled
constexpr uint64_t kWaitCycles = 2000000000ull;  // about one second
constexpr uint32_t kOddScales = 1u << 16;  // beside the bits of the unit's bad boxes
// Units whose marks are told apart. A tile passes over the special units that it has no part in: that no wait of it is a phase
// off takes slots for more units than the ring holds.
constexpr int kFixSlots = 8, kBadSlots = 6;
constexpr int kCountersPerCta = 8;       // a counter for each warp's 32 rows of the two tiles

// Tiles of a block: S and O of one take 128 + DP of the 512 columns of tensor memory.
__host__ __device__ constexpr int tiles_of(int dp) { return dp == 256 ? 1 : 2; }

template <int DP, int CODE>
struct Layout {
  static constexpr bool kCoded = CODE != KL_CODE_NONE;
  // Two softmax warpgroups; load, each tile's products, V; over an 8-bit cache four warps that widen its codes.
  static constexpr int kThreads = kCoded ? 512 : 384;
  // Registers: 256 * 136 + 256 * 120 = 512 * 128, 256 * 176 + 128 * 152 = 384 * 168, the launch's.
  static constexpr int kSoftmaxRegs = kCoded ? 136 : 176, kOtherRegs = kCoded ? 120 : 152;
  static constexpr int kTiles = tiles_of(DP);
  // Of 8 exponentials, those on the multiply-add pipes (a prompt of 8192 tokens: 589 us with none, 571 with 3 in runs of 20
  // calls; 638 and 632 under the power cap). Over codes the warps are short of issue slots (chunks over 8192 tokens: 1,195 us
  // with none, 1,238 with 3).
  static constexpr int kByFma = kCoded ? 0 : 3;
  static constexpr int kHalves = DP / 64;                   // 128-byte column blocks of a 16-bit row
  static constexpr uint32_t kHalf = 128u * 128u;            // 128 rows of one
  static constexpr uint32_t kTile = kHalves * kHalf;
  static constexpr int kStages = DP == 256 ? 2 : kCoded ? (DP == 128 ? 3 : 4) : (DP == 128 ? 5 : 8);
  static constexpr int kRawStages = !kCoded ? 0 : DP == 256 ? 1 : DP == 128 ? 4 : 6;
  static constexpr uint32_t kRawTile = 128u * DP;           // codes, a row after the other
  static constexpr uint32_t kRing = kTiles * kTile;         // Q's tiles first
  static constexpr uint32_t kRaw = kRing + kStages * kTile;
  static constexpr uint32_t kBars = kRaw + kRawStages * kRawTile;
  static constexpr uint32_t kWords = kBars + 384;           // ints
  static constexpr uint32_t kScales = kWords + 256;         // [kBadSlots][K, V, log2 |V|][16]: a scale for every 8 keys
  static constexpr uint32_t kBytes = kScales + (kCoded ? kBadSlots * 3 * 64 : 0) + 1024;  // slack to align the base to 1024 bytes
  // A unit's marks and scales are written before its boxes wait for room: the unit kBadSlots before it has been used then.
  static_assert(2 * kBadSlots >= kStages + kRawStages + 2, "slots of units");
  // Barriers of the rings.
  static constexpr int kFull = 24, kEmpty = kFull + kStages, kRawFull = kEmpty + kStages, kRawEmpty = kRawFull + kRawStages;
  static constexpr int kBarCount = kRawEmpty + kRawStages;
  static_assert(kBarCount * 8 <= 384 && kBytes <= 232448, "shared memory");
};

// Barriers, 8 bytes each from Layout::kBars on.
enum Bar { kQFull0, kQFull1, kQEmpty0, kQEmpty1, kSFull0, kSFull1, kPReady0, kPReady1, kPRest0, kPRest1, kOFull0, kOFull1, kDrain0, kDrain1, kTurn0, kTurn1, kFix0, kFixEnd = kFix0 + kFixSlots };
static_assert(kFixEnd == 24, "the rings' barriers follow");

// Words from Layout::kWords on.
enum Word { kTmem, kDead, kStartSeq, kStartLo, kStartHi, kStartHead, kStartBlock, kStartUnit, kStartFirst, kStartN, kStartLen, kVFlag, kBad = kVFlag + kFixSlots, kScan = kBad + kBadSlots };

struct Smem {
  uint32_t base;        // shared address
  uint8_t* ptr;
  uint32_t bars;
  volatile int* words;
  uint32_t* status;
  __device__ uint32_t bar(int i) const { return bars + 8u * i; }
};

// False when the wait ran out or another one of the CTA has: the role then leaves its loops.
__device__ __forceinline__ bool wait_for(const Smem& sm, uint32_t bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t start = clock64();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i) {
      if (mbar_try_wait(bar, parity)) return true;
    }
    if (sm.words[kDead]) return false;
    if (static_cast<uint64_t>(clock64()) - start > kWaitCycles) {
      atomicOr(sm.status, kStatusWaitTimeout);
      sm.words[kDead] = 1;
      return false;
    }
  }
}

// ----------------------------------------------------------------- plan

// Units of row block k of sequence s: the keys that its last row sees, at least one unit.
__device__ __forceinline__ int block_units(const Args& a, const Seq& s, int k) {
  const int rows_end = min(s.n, (k + 1) * a.block_tokens);
  return max(1, (keys_of(a, s, rows_end - 1) + kBN - 1) / kBN);
}

__device__ __forceinline__ int blocks_of(const Args& a, const Seq& s) { return (s.n + a.block_tokens - 1) / a.block_tokens; }

// The same summed over a sequence's blocks. Causal, all but the last block, step = tokens of a block:
//   max(1, ceil((base + (k + 1) step) / 128)), base = len - n,
// is 1 while base + (k + 1) step <= 128 and floor((A + i step) / 128) after that. The sum of the latter is that of the
// terms less that of their remainders, over 128; the remainders run through the residues of A mod g, g = gcd(step, 128).
__device__ __forceinline__ int64_t head_units(const Args& a, const Seq& s) {
  const int nb = blocks_of(a, s);
  if (nb == 0) return 0;
  if (!a.causal) return static_cast<int64_t>(nb) * max(1, (s.len + kBN - 1) / kBN);
  const int step = a.block_tokens, base = s.len - s.n;
  int64_t total = max(1, (s.len + kBN - 1) / kBN);
  const int ones = min(nb - 1, base <= kBN - step ? (kBN - base) / step : 0);
  const int64_t m = nb - 1 - ones;
  total += ones;
  if (m > 0) {
    const int64_t A = base + static_cast<int64_t>(ones + 1) * step + kBN - 1;
    const int g = min(step & -step, kBN), p = kBN / g;
    int64_t rest = (m / p) * (p * (A % g) + static_cast<int64_t>(g) * p * (p - 1) / 2);
    int r = static_cast<int>(A % kBN);
    for (int i = 0; i < m % p; ++i) {
      rest += r;
      r = (r + step) % kBN;
    }
    total += (m * A + step * (m * (m - 1) / 2) - rest) / kBN;
  }
  return total;
}

struct Segment {
  Seq s;
  int b, h, blk;   // sequence, KV head, row block
  int j0, j1, nt;  // its units of this segment, and how many the block has
  int64_t first;   // number of the block's first unit
};

__device__ __forceinline__ Seq start_seq(const Smem& sm) {
  return Seq{sm.words[kStartFirst], sm.words[kStartN], sm.words[kStartLen]};
}

struct Walk {
  Seq s;
  int b, h, blk, j, nb;
  int64_t u, u1;

  // At the place that find_start left.
  __device__ void init(const Args& a, const Smem& sm, int64_t u_first, int64_t u_end) {
    u = u_first;
    u1 = u_end;
    b = sm.words[kStartSeq];
    h = sm.words[kStartHead];
    blk = sm.words[kStartBlock];
    j = sm.words[kStartUnit];
    s = start_seq(sm);
    nb = blocks_of(a, s);
  }

  __device__ bool next(const Args& a, Segment& g) {
    if (u >= u1) return false;
    const int nt = block_units(a, s, blk);
    const int take = static_cast<int>(min(u1 - u, static_cast<int64_t>(nt - j)));
    g = Segment{s, b, h, blk, j, j + take, nt, u - j};
    u += take;
    j += take;
    if (j == nt && u < u1) {
      j = 0;
      if (++blk == nb) {
        blk = 0;
        if (++h == a.hkv) {
          h = 0;
          do {
            s = read_seq(a, ++b, false);
          } while (s.n == 0 && b + 1 < a.batch);
          nb = blocks_of(a, s);
        }
      }
    }
    return true;
  }
};

// Where unit `off` of sequence b lies, by a whole warp.
__device__ __forceinline__ void find_start(const Args& a, const Smem& sm, int lane) {
  const Seq s = start_seq(sm);
  int64_t off = static_cast<int64_t>(static_cast<uint32_t>(sm.words[kStartLo])) | (static_cast<int64_t>(sm.words[kStartHi]) << 32);
  const int64_t per_head = head_units(a, s);
  const int h = static_cast<int>(off / per_head), nb = blocks_of(a, s);
  off -= h * per_head;
  int blk = 0;
  for (;;) {  // 32 blocks at a time
    const int k = blk + lane;
    int inc = k < nb ? block_units(a, s, k) : 0;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, m);
      if (lane >= m) inc += y;
    }
    const int passed = __popc(__ballot_sync(0xffffffffu, inc <= off && k < nb));
    if (passed < 32 || blk + 32 >= nb) {
      const int before = __shfl_sync(0xffffffffu, inc, max(0, passed - 1));
      if (passed > 0) off -= before;
      blk += passed;
      break;
    }
    off -= __shfl_sync(0xffffffffu, inc, 31);
    blk += 32;
  }
  if (lane == 0) {
    sm.words[kStartHead] = h;
    sm.words[kStartBlock] = blk;
    sm.words[kStartUnit] = static_cast<int>(off);
  }
}

// What a block's tile t has to do within a segment: units [j0, end(t)).
struct Tiles {
  int tok0_, end0, end1;
  int step;        // tokens of a tile
  int seen_first;  // keys that the block's first row sees
  __device__ Tiles(const Args& a, const Segment& g) : tok0_(g.blk * a.block_tokens), step(a.tile_tokens) {
    end0 = end_of(a, g, 0);
    end1 = a.block_tokens > step ? end_of(a, g, 1) : g.j0;
    seen_first = keys_of(a, g.s, tok0_);
  }
  __device__ int tok0(int t) const { return tok0_ + t * step; }    // first token of the tile
  __device__ int end(int t) const { return t ? end1 : end0; }      // end of its units in the segment
  __device__ int end_of(const Args& a, const Segment& g, int t) const {
    int nt = 0;
    if (tok0(t) < g.s.n) nt = max(1, (keys_of(a, g.s, min(g.s.n, tok0(t) + step) - 1) + kBN - 1) / kBN);
    return max(g.j0, min(g.j1, nt));
  }
  // Units in which some row does not see every key.
  __device__ bool special(int j) const { return (j + 1) * kBN > seen_first; }
};

// ----------------------------------------------------------------- PTX

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, int x, int y, int z, int w, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar), "l"(policy)
      : "memory");
}

// The products are issued by one thread, and a chain of 64-bit shifts before each of them would hold them up: a
// descriptor's low word moves by the offset in 16-byte units, its high word is a constant.
__device__ __forceinline__ uint64_t desc_of(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4 << 16); }
// Bytes between groups of 8 rows, version, 128-byte swizzle.
__device__ __forceinline__ uint32_t desc_hi(uint32_t sbo) { return sbo >> 4 | (1u << 14) | (2u << 29); }

// D[tmem] (+)= A[tmem] . B[smem]; A's row i is lane i, two 16-bit elements a column.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  const uint32_t none = 0u;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(none)
      : "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t addr, float (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const float (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "f"(r[0]), "f"(r[1]),
               "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7])
               : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}

__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of a pair on the multiply-add pipes, x <= 15 (NaN is not kept): 2^n 2^f with n the nearest whole number, f in [-1/2, 1/2],
// and 2^f by 1 + c1 f + c2 f^2 + ..., the coefficients of least relative error (by linear programming over [-1/2, 1/2]):
// 1.02e-4 with three of them (P in bf16, half a step 2^-8), 3.0e-6 with four (fp16, 2^-11). Zero from x = -127 down, exactly.
template <int DEGREE>
__device__ __forceinline__ void exp2_pair(uint64_t x2, float& p0, float& p1) {
  float x0, x1;
  unpair(x2, x0, x1);
  const uint64_t x = pair(fmaxf(x0, -127.0f), fmaxf(x1, -127.0f));
  const uint64_t shifter = pair(12582912.0f, 12582912.0f), back = pair(-12582912.0f, -12582912.0f);  // 1.5 * 2^23
  const uint64_t n = add2(x, shifter);  // n in the low bits
  const uint64_t minus = pair(-1.0f, -1.0f);
  const uint64_t f = fma2(add2(n, back), minus, x);
  uint64_t y;
  if (DEGREE == 3) {
    y = fma2(pair(0.05500893294811249f, 0.05500893294811249f), f, pair(0.2422109693288803f, 0.2422109693288803f));
    y = fma2(y, f, pair(0.6932829022407532f, 0.6932829022407532f));
  } else {
    y = fma2(pair(0.009585382416844368f, 0.009585382416844368f), f, pair(0.05590662732720375f, 0.05590662732720375f));
    y = fma2(y, f, pair(0.24024038016796112f, 0.24024038016796112f));
    y = fma2(y, f, pair(0.6931241750717163f, 0.6931241750717163f));
  }
  y = fma2(y, f, pair(1.0f, 1.0f));
  float n0, n1, y0, y1;
  unpair(n, n0, n1);
  unpair(y, y0, y1);
  p0 = __uint_as_float((__float_as_uint(n0) << 23) + __float_as_uint(y0));
  p1 = __uint_as_float((__float_as_uint(n1) << 23) + __float_as_uint(y1));
}
// 32 bytes a lane in one store: a whole sector.
__device__ __forceinline__ void store32(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// ----------------------------------------------------------------- pieces of cut blocks

// CTA c's piece of a block that an earlier CTA began lies in slot 2c, of one that it began itself in slot 2c + 1.
// A slot: for each tile O [128][DP] fp32, then maxima [128] and sums [128].
template <int DP>
__device__ __forceinline__ float* piece_at(const Args& a, int64_t slot, int t) {
  return a.partials + (slot * tiles_of(DP) + t) * (static_cast<int64_t>(DP) + 2) * 128;
}

template <typename V>
__device__ __forceinline__ V load_cg(const float* p) {
  V v;
  if constexpr (sizeof(V) == 16) {
    const float4 f = __ldcg(reinterpret_cast<const float4*>(p));
    v.v[0] = f.x, v.v[1] = f.y, v.v[2] = f.z, v.v[3] = f.w;
  } else {
    const float2 f = __ldcg(reinterpret_cast<const float2*>(p));
    v.v[0] = f.x, v.v[1] = f.y;
  }
  return v;
}

// ----------------------------------------------------------------- roles

struct Plan {
  int64_t total;
  int runs;
  __device__ int64_t begin(int c) const { return total * c / runs; }
  __device__ int run_of(int64_t u) const { return static_cast<int>(((u + 1) * runs - 1) / total); }
};

template <typename T, int DP, int CODE>
__device__ __forceinline__ void load_role(const Args& a, const Smem& sm, Walk w, int lane, const CUtensorMap* mq, const CUtensorMap* mk,
                                          const CUtensorMap* mv) {
  using L = Layout<DP, CODE>;
  const uint64_t keep = l2_policy_evict_normal(), once = l2_policy_evict_first();
  constexpr int kDepth = L::kCoded ? L::kRawStages : L::kStages;
  constexpr int kFull = L::kCoded ? L::kRawFull : L::kFull, kEmpty = L::kCoded ? L::kRawEmpty : L::kEmpty;
  const int boxes = kBN / a.box_rows;
  const uint32_t box_bytes = a.box_rows * (L::kCoded ? DP : 128u);
  uint32_t slot = 0, phase = 0, issued = 0, unit = 0;
  uint32_t q_loads = 0;
  bool ok = true;
  Segment g{};
  // Lane i looks after box i of a unit: its page, num_pages (for zeros) past the sequence's end or where the id is
  // no page's. Ids are asked for two units ahead, scales one.
  auto page_of = [&](int j) -> int64_t {
    const int tok = j * kBN + lane * a.box_rows;
    return j < g.j1 && lane < boxes && tok < g.s.len ? __ldcg(a.block_table + g.b * a.bt_stride + tok / a.page_size) : a.num_pages;
  };
  auto scale_of = [&](const float* scales, int64_t page) {
    return L::kCoded && page >= 0 && page < a.num_pages ? __ldcg(scales + page * a.scale_stride + g.h) : 0.0f;
  };
  auto load_q = [&](const Segment& g, const Tiles& tiles) {  // lane t: tile t
    if (lane < 2 && tiles.end(lane) > g.j0) {
      if (q_loads > 0) ok = wait_for(sm, sm.bar(kQEmpty0 + lane), (q_loads - 1) & 1);
      ++q_loads;
      if (ok) {
        mbar_arrive_expect_tx(sm.bar(kQFull0 + lane), L::kHalves * a.tile_tokens * a.group * 128u);
#pragma unroll
        for (int c = 0; c < L::kHalves; ++c) {
          tma_load_3d(sm.base + lane * L::kTile + c * L::kHalf, mq, c * 64, g.h * a.group, static_cast<int>(g.s.first) + tiles.tok0(lane),
                      sm.bar(kQFull0 + lane), once);
        }
      }
    }
    ok = __all_sync(0xffffffffu, ok);
  };
  bool first_segment = true;
  while (ok && w.next(a, g)) {
    const Tiles tiles(a, g);
    int64_t page = page_of(g.j0), page1 = page_of(g.j0 + 1);
    if (first_segment) load_q(g, tiles);
    float ks = scale_of(a.k_scale, page), vs = scale_of(a.v_scale, page);
    for (int j = g.j0; ok && j < g.j1; ++j, ++unit) {
      const int64_t page2 = page_of(j + 2);
      const float ks1 = scale_of(a.k_scale, page1), vs1 = scale_of(a.v_scale, page1);
      const int tok = j * kBN + lane * a.box_rows;
      const bool bad = lane < boxes && tok < g.s.len && (page < 0 || page >= a.num_pages);
      if (bad) page = a.num_pages;
      const uint32_t bad_boxes = __ballot_sync(0xffffffffu, bad);
      // Scales that are negative, infinite or NaN.
      const bool odd = L::kCoded && __any_sync(0xffffffffu, !(ks >= 0.0f && ks < INFINITY && vs >= 0.0f && vs < INFINITY));
      if (lane == 0) {
        sm.words[kBad + unit % kBadSlots] = static_cast<int>(bad_boxes | (odd ? kOddScales : 0u));
        if (bad_boxes) atomicOr(sm.status, kStatusBadPage);
      }
      if constexpr (L::kCoded) {
        const int from = (lane & 15) * 8 >> a.box_shift;
        const float x = __shfl_sync(0xffffffffu, ks, from), y = __shfl_sync(0xffffffffu, vs, from);
        float* const to = reinterpret_cast<float*>(sm.ptr + L::kScales) + unit % kBadSlots * 48 + lane;
        *to = lane < 16 ? x * a.scale_log2 : y;
        if (std::is_same<T, __half>::value && lane < 16) to[32] = __log2f(fabsf(y));
      }
      __syncwarp();
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t full = sm.bar(kFull + slot), empty = sm.bar(kEmpty + slot);
        if (issued >= kDepth) ok = wait_for(sm, empty, phase ^ 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(full, L::kCoded ? L::kRawTile : L::kTile);
        __syncwarp();
        if (lane < boxes) {
          if constexpr (L::kCoded) {
            tma_load_4d(sm.base + L::kRaw + slot * L::kRawTile + lane * box_bytes, kv ? mv : mk, 0, g.h, tok % a.page_size,
                        static_cast<int>(page), full, keep);
          } else {
            const uint32_t to = sm.base + L::kRing + slot * L::kTile;
            if (a.merged) {
              const int group = page < a.num_pages ? static_cast<int>(page) * a.page_groups + g.h * a.head_groups + tok % a.page_size / 8
                                                   : a.total_groups;
              tma_load_4d(to + (lane << a.box_shift >> 3) * a.group_bytes, kv ? mv : mk, 0, 0, g.h * a.head_halves, group, full, keep);
            } else {
#pragma unroll
              for (int c = 0; c < L::kHalves; ++c) {
                tma_load_4d(to + c * L::kHalf + lane * box_bytes, kv ? mv : mk, c * 64, g.h, tok % a.page_size, static_cast<int>(page), full,
                            keep);
              }
            }
          }
        }
        ++issued;
        if (++slot == kDepth) {
          slot = 0;
          phase ^= 1;
        }
        // Later segments' Q behind their first keys, which need not wait for its room.
        if (kv == 0 && j == g.j0 && !first_segment) load_q(g, tiles);
        if (!ok) break;
      }
      first_segment = false;
      page = page1;
      page1 = page2;
      ks = ks1;
      vs = vs1;
    }
  }
  // Nothing may be in flight into this CTA's shared memory when it ends; normally it has long landed.
  if (lane < 2 && q_loads > 0) {
    const uint64_t start = clock64();
    while (!mbar_try_wait(sm.bar(kQFull0 + lane), (q_loads - 1) & 1) && static_cast<uint64_t>(clock64()) - start < kWaitCycles) {
    }
  }
  if (lane == 0) {
    for (uint32_t k = 0; k < min(issued, static_cast<uint32_t>(kDepth)); ++k) {
      const uint32_t i = issued - 1 - k, s = i % kDepth;
      const uint64_t start = clock64();
      while (!mbar_try_wait(sm.bar(kFull + s), (i / kDepth) & 1) && static_cast<uint64_t>(clock64()) - start < kWaitCycles) {
      }
    }
  }
  __syncwarp();
}

// ----------------------------------------------------------------- codes to 16 bits

// Two codes, the bytes 2 * HI and 2 * HI + 1 of a word, as a pair of TO; exact: e4m3 has 4 significant bits, int8 7.
template <typename TO, int CODE, int HI>
__device__ __forceinline__ uint32_t widen_pair(uint32_t w) {
  if constexpr (CODE == KL_CODE_E4M3) {
    const uint32_t h = HI ? e4m3x2_hi_to_f16x2(w) : e4m3x2_lo_to_f16x2(w);
    if constexpr (std::is_same<TO, __half>::value) return h;
    const float2 f = Storage<__half>::unpack2(h);
    return Storage<__nv_bfloat16>::pack2(f.x, f.y);
  } else if constexpr (std::is_same<TO, __half>::value) {
    // The code with its sign bit turned over, as the last bits of 1024 + (code + 128).
    const uint32_t x = __byte_perm(w ^ 0x80808080u, 0x64646464u, HI ? 0x7372 : 0x7170);
    const __half2 bias = __floats2half2_rn(1152.0f, 1152.0f);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), bias);
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    // 128 + the low seven bits, less 256 for a negative code and 128 for another.
    const uint32_t x = __byte_perm(w, 0u, HI ? 0x4342 : 0x4140);
    const uint32_t p = (x & 0x007f007fu) | 0x43004300u, n = (x & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&p), *reinterpret_cast<const __nv_bfloat162*>(&n));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// One row of a tile: codes in, 16-bit elements in the 128-byte swizzle out. The rows of a warp start at different
// places of their row, which leaves neither side with bank conflicts.
template <typename TO, int DP, int CODE>
__device__ __forceinline__ void widen_row(uint32_t raw, uint32_t tile, int row) {
  using L = Layout<DP, CODE>;
  constexpr int kUnits = DP / 16;
#pragma unroll 2
  for (int k = 0; k < kUnits; ++k) {
    const int u = (k + row) & (kUnits - 1);
    const uint4 v = lds128(raw + row * DP + u * 16);
    const uint32_t in[4] = {v.x, v.y, v.z, v.w};
    uint32_t out[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = widen_pair<TO, CODE, 0>(in[i]);
      out[2 * i + 1] = widen_pair<TO, CODE, 1>(in[i]);
    }
    const uint32_t at = tile + (u >> 2) * L::kHalf + row * 128u;  // groups of 8 rows 1024 bytes apart, halves kHalf
    const uint32_t c = (2 * u) & 7, s = row & 7;
    sts128(at + ((c ^ s) << 4), make_uint4(out[0], out[1], out[2], out[3]));
    sts128(at + (((c + 1) ^ s) << 4), make_uint4(out[4], out[5], out[6], out[7]));
  }
}

// Four warps, a thread a row.
template <typename T, int DP, int CODE>
__device__ __forceinline__ void widen_role(const Args& a, const Smem& sm, Walk w, int row) {
  using L = Layout<DP, CODE>;
  uint32_t raw_slot = 0, raw_phase = 0, slot = 0, phase = 0;
  const int64_t items = 2 * (w.u1 - w.u);
  for (int64_t i = 0; i < items; ++i) {
    bool ok = wait_for(sm, sm.bar(L::kRawFull + raw_slot), raw_phase);
    if (i >= L::kStages) ok = ok && wait_for(sm, sm.bar(L::kEmpty + slot), phase ^ 1);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) return;
    const uint32_t raw = sm.base + L::kRaw + raw_slot * L::kRawTile, tile = sm.base + L::kRing + slot * L::kTile;
    widen_row<T, DP, CODE>(raw, tile, row);
    fence_proxy_async_smem();
    __syncwarp();
    if ((row & 31) == 0) {
      mbar_arrive(sm.bar(L::kFull + slot));
      mbar_arrive(sm.bar(L::kRawEmpty + raw_slot));
    }
    if (++raw_slot == L::kRawStages) {
      raw_slot = 0;
      raw_phase ^= 1;
    }
    if (++slot == L::kStages) {
      slot = 0;
      phase ^= 1;
    }
  }
}

// A value that is the same in all lanes, known to be so: operands of the products live in uniform registers, and moving
// them there one by one for a lone thread took as long as the products (a unit's 4 products of 128 x 128 x 128: 3500 cycles).
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}

// A warp for each tile t; one thread of it issues.
template <typename T, int DP, int CODE>
__device__ __forceinline__ void mma_role(const Args& a, const Smem& sm, Walk w, int t, uint32_t tmem) {
  using L = Layout<DP, CODE>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = umma_idesc_f16(BF16, 128, kBN, false), IDESC_O = umma_idesc_f16(BF16, 128, DP, true);
  const int ksteps = (a.dim + 15) / 16;
  const uint32_t sq = uniform(desc_lo(sm.base + t * L::kTile, 16)), ring = uniform(desc_lo(sm.base + L::kRing, 0));
  const uint32_t hi = desc_hi(a.group_bytes);
  const uint32_t s_at = uniform(tmem + t * 128), o_at = uniform(tmem + 256 + t * 128);
  uint32_t slot = 0, phase = 0, unit = 0, q_phase = 0, p_phase = 0, turn = 0;
  bool ok = true;
  Segment g{};
  auto wait = [&](uint32_t bar, uint32_t parity) {
    ok = ok && wait_for(sm, bar, parity);
    ok = __all_sync(0xffffffffu, ok);
  };
  auto commit = [&](uint32_t bar) {
    if (elect_one()) umma_commit(bar);
  };
  // Waits for a stage; gives it back when the products issued so far are done.
  auto ring_wait = [&] { wait(sm.bar(L::kFull + slot), phase); };
  auto ring_next = [&] {
    commit(sm.bar(L::kEmpty + slot));
    if (++slot == L::kStages) {
      slot = 0;
      phase ^= 1;
    }
  };
  // The tiles take turns, unit by unit: two threads' products would share the tensor cores evenly, and both tiles' softmax
  // would then run at once and wait at once.
  auto my_turn = [&] {
    if (t == 1 || turn > 0) wait(sm.bar(kTurn0 + t), (t == 1 ? turn : turn - 1) & 1);
  };
  auto scores = [&](uint32_t k_slot) {
    const uint32_t sk = uniform(ring + k_slot * (L::kTile >> 4) + (1u << 16));
    if (elect_one()) {
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        const uint32_t in_half = (ks % 4) * 32u >> 4;
        if (ks < ksteps) {
          umma_f16(s_at, desc_of(sq + ((ks / 4) * L::kHalf >> 4) + in_half, desc_hi(1024)), desc_of(sk + (ks / 4) * (a.half_bytes >> 4) + in_half, hi),
                   IDESC_S, ks > 0);
        }
      }
      umma_commit(sm.bar(kSFull0 + t));
    }
    __syncwarp();
  };
  while (ok && w.next(a, g)) {
    const Tiles tiles(a, g);
    const int end = tiles.end(t);
    ring_wait();
    if (end > g.j0) {
      wait(sm.bar(kQFull0 + t), q_phase);
      q_phase ^= 1;
      if (!ok) break;
      tcgen05_fence_after();
      scores(slot);
      if (end == g.j0 + 1) commit(sm.bar(kQEmpty0 + t));
    }
    if (!ok) break;
    ring_next();
    for (int j = g.j0; ok && j < g.j1; ++j, ++unit) {
      // V of this unit and K of the next one before P: what follows P is then issued without a pause.
      const uint32_t v_slot = slot, k_slot = v_slot + 1 == L::kStages ? 0 : v_slot + 1;
      const bool more_keys = j + 1 < g.j1;
      ring_wait();
      if (more_keys) wait(sm.bar(L::kFull + k_slot), k_slot == 0 ? phase ^ 1 : phase);
      if (j < end) {
        const uint32_t sv = uniform(ring + v_slot * (L::kTile >> 4) + (a.half_bytes >> 4 << 16)), again = uniform(j > g.j0);
        const bool special = tiles.special(j);
        bool by_hand = false;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          wait(sm.bar((half ? kPRest0 : kPReady0) + t), p_phase);
          if (half == 0) my_turn();
          if (!ok) break;
          tcgen05_fence_after();
          if (half == 0) by_hand = special && sm.words[kVFlag + unit % kFixSlots];
          if (!by_hand && elect_one()) {
#pragma unroll
            for (int ks = half * kBN / 32; ks < (half + 1) * kBN / 32; ++ks) {
              umma_f16_ts(o_at, s_at + ks * 8, desc_of(sv + ks * (a.group_bytes >> 3), hi), IDESC_O, ks > 0 ? 1u : again);
            }
          }
          __syncwarp();
        }
        p_phase ^= 1;
        if (!ok) break;
        if (j + 1 < end) {
          scores(k_slot);
          if (j + 2 == end) commit(sm.bar(kQEmpty0 + t));
        } else {
          commit(sm.bar(kOFull0 + t));
        }
      } else {
        my_turn();
      }
      if (!ok) break;
      if (elect_one()) mbar_arrive(sm.bar(kTurn0 + (1 - t)));
      ++turn;
      ring_next();  // V and, if there are more keys, K
      if (more_keys) ring_next();
    }
  }
  // Every product has ended before the CTA does.
  commit(sm.bar(kDrain0 + t));
  const uint64_t start = clock64();
  while (!mbar_try_wait(sm.bar(kDrain0 + t), 0) && static_cast<uint64_t>(clock64()) - start < kWaitCycles) {
  }
  __syncwarp();
}

// Where half `half` of row `row` lies in a tile.
__device__ __forceinline__ uint32_t row_at(const Args& a, int row, int half) {
  return (row >> 3) * a.group_bytes + half * a.half_bytes + (row & 7) * 128u;
}

// One warp: the V rows of special units.
template <typename T, int DP, int CODE>
__device__ __forceinline__ void fix_role(const Args& a, const Smem& sm, Walk w, int lane) {
  using L = Layout<DP, CODE>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kExp = BF16 ? 0x7f807f80u : 0x7c007c00u, kOne = BF16 ? 0x00800080u : 0x04000400u;
  uint32_t unit = 0;
  bool ok = true;
  Segment g{};
  while (ok && w.next(a, g)) {
    const Tiles tiles(a, g);
    for (int j = g.j0; ok && j < g.j1; ++j, ++unit) {
      // Every stage is waited for and given back: a wait by parity must not be more than a phase off.
      uint32_t slot = 0;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t i = 2 * unit + kv;
        slot = i % L::kStages;
        ok = ok && wait_for(sm, sm.bar(L::kFull + slot), (i / L::kStages) & 1);
        if (kv == 0 && lane == 0) mbar_arrive(sm.bar(L::kEmpty + slot));
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint32_t empty = sm.bar(L::kEmpty + slot);
      if (!tiles.special(j)) {
        if (lane == 0) mbar_arrive(empty);
        continue;
      }
      const uint32_t sv = sm.base + L::kRing + slot * L::kTile;
      const int held = max(0, min(kBN, g.s.len - j * kBN));                            // rows of tokens
      const int boxed = min(kBN, (held + a.box_rows - 1) / a.box_rows * a.box_rows);   // zeros from here on
      const int unseen = max(0, min(held, tiles.seen_first - j * kBN));                // seen by all below
      for (int k = lane; k < (boxed - held) * L::kHalves * 8; k += 32) {
        const int row = held + k / (L::kHalves * 8), c = k / 8 % L::kHalves, u = k % 8;
        sts128(sv + row_at(a, row, c) + u * 16u, make_uint4(0u, 0u, 0u, 0u));
      }
      uint32_t odd = 0;
      for (int k = lane; k < (held - unseen) * L::kHalves * 8; k += 32) {
        const int row = unseen + k / (L::kHalves * 8), c = k / 8 % L::kHalves, u = k % 8;
        const uint4 v = lds128(sv + row_at(a, row, c) + u * 16u);
        odd |= ((v.x & kExp) + kOne) | ((v.y & kExp) + kOne) | ((v.z & kExp) + kOne) | ((v.w & kExp) + kOne);
      }
      odd = __any_sync(0xffffffffu, (odd & 0x80008000u) != 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        // Scales that are no numbers are taken by hand, too: a masked probability times one would be NaN.
        sm.words[kVFlag + unit % kFixSlots] = static_cast<int>(odd | (static_cast<uint32_t>(sm.words[kBad + unit % kBadSlots]) & kOddScales));
        mbar_arrive(sm.bar(kFix0 + unit % kFixSlots));
        mbar_arrive(empty);
      }
      __syncwarp();
    }
  }
}

template <typename T, int DP, int CODE>
__device__ __forceinline__ void softmax_role(const Args& a, const Smem& sm, Walk w, const Plan& plan, int t, int warp, int lane, uint32_t tmem) {
  using L = Layout<DP, CODE>;
  const int row = warp * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
  const uint32_t tS = tmem + lanes + t * 128, tO = tmem + lanes + 256 + t * 128;
  const float sl = a.scale_log2;
  const uint64_t sl2 = pair(sl, sl);
  // fp16 probabilities (and their sum) are held 2^7 times as large, at most 2^15 with kLazy: those below 2^-14 of a row's
  // largest would lose bits to fp16's subnormals (16,000 keys of weight 2^-22 beside one of 1: 2 % of their share).
  constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
  // Over codes P holds probabilities times value scales. bf16 has the range for any of them. In fp16 they are relative to a row's
  // largest such product so far, 2^w_ref, which follows it as m follows the scores; O is then in units of 2^(w_ref - kLift), l
  // in those of 2^m.
  constexpr bool kWeighted = L::kCoded && std::is_same<T, __half>::value;
  uint32_t unit = 0, s_phase = 0, o_phase = 0, fix_phases = 0;
  bool ok = true;
  Segment g{};
  while (ok && w.next(a, g)) {
    const Tiles tiles(a, g);
    const int tok = row / a.group, head = row - tok * a.group;
    const bool valid = row < a.tile_tokens * a.group && tiles.tok0(t) + tok < g.s.n;
    const int limit = valid ? keys_of(a, g.s, tiles.tok0(t) + tok) : 0;
    float m = -INFINITY, l = 0.0f, w_ref = -INFINITY;
    uint32_t u = unit;
    for (int j = g.j0; j < g.j1; ++j, ++u) {
      const bool special = tiles.special(j);
      const uint32_t fix = u % kFixSlots;
      if (j >= tiles.end(t)) {  // the other tile's units: only the count of special ones goes on
        if (special) fix_phases ^= 1u << fix;
        continue;
      }
      ok = wait_for(sm, sm.bar(kSFull0 + t), s_phase);
      s_phase ^= 1;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tcgen05_fence_after();
      const uint32_t marks = static_cast<uint32_t>(sm.words[kBad + u % kBadSlots]);
      const int cols = limit - j * kBN;  // columns that this row sees
      const float* const scales = reinterpret_cast<const float*>(sm.ptr + L::kScales) + u % kBadSlots * 48;
      const bool plain = !special && marks == 0;
      if (!plain) {
        // S is put back as scaled, and -inf where masked: what follows need not ask.
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t s[32];
          tmem_ld32(tS + c, s);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (L::kCoded) s[i] = __float_as_uint(__uint_as_float(s[i]) * scales[(c + i) / 8]);
            if (c + i >= cols || (marks >> ((c + i) >> a.box_shift) & 1u)) s[i] = 0xff800000u;
          }
          tmem_st32(tS + c, s);
        }
        tmem_wait_st();
      }
      // The row's maximum. Rolled loops here and below: longer code would not stay in the instruction caches.
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, wx = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < 128; c += 64) {
        uint32_t s[2][32];
        tmem_ld32(tS + c, s[0]);
        tmem_ld32(tS + c + 32, s[1]);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          float top = L::kCoded ? -INFINITY : mx[q & 3];
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            top = max3(top, __uint_as_float(s[q / 4][q % 4 * 8 + i]), __uint_as_float(s[q / 4][q % 4 * 8 + i + 1]));
          }
          if constexpr (L::kCoded) {
            top *= plain ? scales[c / 8 + q] : 1.0f;  // no scale is negative here
            // A masked group's value scale does not count, whatever it is.
            if constexpr (kWeighted) wx = max3(wx, wx, top == -INFINITY ? top : top + scales[32 + c / 8 + q]);
            top = max3(mx[q & 3], mx[q & 3], top);
          }
          mx[q & 3] = top;
        }
      }
      const float mc = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * (L::kCoded ? 1.0f : sl);
      float alpha = 1.0f;
      if (!(mc <= m + kLazy)) {
        // 0 where m is -inf. An infinite or NaN score makes the row NaN, by way of m: exp2_pair does not keep NaN.
        alpha = mc < INFINITY ? exp2_approx(m - mc) : NAN;
        m = mc < INFINITY ? mc : NAN;
        l *= alpha;
      }
      float p_scale = 1.0f;
      if constexpr (kWeighted) {
        alpha = 1.0f;
        if (!(wx <= w_ref + kLazy)) {
          alpha = wx < INFINITY ? exp2_approx(w_ref - wx) : NAN;
          w_ref = wx < INFINITY ? wx : NAN;
        }
        p_scale = exp2_approx(fminf(m - w_ref + kLift, 127.0f));
      }
      if (j > g.j0 && __any_sync(0xffffffffu, !(alpha >= 1.0f))) {
        // S of this unit is complete, and so is O += P V of the one before.
#pragma unroll 1
        for (int c = 0; c < DP; c += 8) {
          float o[8];
          tmem_ld8(tO + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] *= alpha;
          tmem_st8(tO + c, o);
        }
      }
      const float shift = (m == -INFINITY ? 0.0f : m) - (kWeighted ? 0.0f : kLift);
      const uint64_t sh2 = pair(-shift, -shift);
      uint64_t sum[2] = {0, 0};
      // P, 32 columns at a time, over columns of S that have been read; the products with the first 64 keys may begin
      // before the rest is done.
      auto put_p = [&](const uint32_t(&s)[16], int c) {
        uint32_t p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint64_t x2 = pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
          float f = 1.0f;
          if constexpr (L::kCoded) f = plain ? scales[c / 8 + i / 4] : 1.0f;
          float x0, x1;
          const uint64_t e2 = fma2(x2, L::kCoded ? pair(f, f) : sl2, sh2);
          if (i * L::kByFma % 8 < L::kByFma) {
            exp2_pair<std::is_same<T, __half>::value ? 4 : 3>(e2, x0, x1);
          } else {
            unpair(e2, x0, x1);
            x0 = exp2_approx(x0);
            x1 = exp2_approx(x1);
          }
          const uint64_t p2 = pair(x0, x1);
          sum[i & 1] = add2(sum[i & 1], p2);
          if constexpr (L::kCoded) {
            float v = scales[16 + c / 8 + i / 4];
            // Finite beside a probability of zero, whatever the scale of the group.
            if constexpr (kWeighted) v = fmaxf(fminf(v * p_scale, 3.0e38f), -3.0e38f);
            unpair(mul2(p2, pair(v, v)), x0, x1);
          }
          p[i] = Storage<T>::pack2(x0, x1);
        }
        tmem_st8(tS + c / 2, p);
      };
      uint32_t s0[16], s1[16];
      tmem_ld16(tS, s0);
#pragma unroll 1
      for (int c = 0; c < 128; c += 32) {
        tmem_wait_ld();
        tmem_ld16(tS + c + 16, s1);
        put_p(s0, c);
        tmem_wait_ld();
        tmem_ld16(tS + (c + 32) % 128, s0);  // the last round's is not used
        put_p(s1, c + 16);
        if (c == 32 && !special) {
          tmem_wait_st();
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(sm.bar(kPReady0 + t));
        }
      }
      tmem_wait_ld();
      {
        float x0, x1;
        unpair(add2(sum[0], sum[1]), x0, x1);
        l += x0 + x1;
      }
      if (special) {
        ok = wait_for(sm, sm.bar(kFix0 + fix), (fix_phases >> fix) & 1u);
        fix_phases ^= 1u << fix;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (sm.words[kVFlag + fix]) {
          // Infinities or NaN in rows of V that not every row sees: P V key by key.
          const uint32_t sv = sm.base + L::kRing + (2 * u + 1) % L::kStages * L::kTile;
          tmem_wait_st();
#pragma unroll 1
          for (int c8 = 0; c8 < DP / 8; ++c8) {
            float o[8];
            tmem_ld8(tO + c8 * 8, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = j > g.j0 ? o[i] : 0.0f;
#pragma unroll 1
            for (int c0 = 0; c0 < kBN; c0 += 16) {
              float pp[8];  // 16 keys' probabilities, in pairs
              tmem_ld8(tS + c0 / 2, pp);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const int c = c0 + k;
                const uint4 v = lds128(sv + row_at(a, c, c8 / 8) + static_cast<uint32_t>(((c8 & 7) ^ (c & 7)) * 16));
                const bool seen = c < cols && !(marks >> (c >> a.box_shift) & 1u);
                const float2 p2 = Storage<T>::unpack2(__float_as_uint(pp[k / 2]));
                const float p = k & 1 ? p2.y : p2.x;
                const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 f = Storage<T>::unpack2(vw[i]);
                  if (seen) {
                    o[2 * i] = fmaf(p, f.x, o[2 * i]);
                    o[2 * i + 1] = fmaf(p, f.y, o[2 * i + 1]);
                  }
                }
              }
            }
            tmem_st8(tO + c8 * 8, o);
          }
        }
      }
      tmem_wait_st();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (special) mbar_arrive(sm.bar(kPReady0 + t));
        mbar_arrive(sm.bar(kPRest0 + t));
      }
    }
    unit += g.j1 - g.j0;
    if (!ok) break;

    // ---- the segment's rows: final, or a piece of a cut block
    const bool active = tiles.end(t) > g.j0;
    if (active) {
      ok = wait_for(sm, sm.bar(kOFull0 + t), o_phase);
      o_phase ^= 1;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tcgen05_fence_after();
    }
    if (t >= L::kTiles || tiles.tok0(t) >= g.s.n) continue;  // no rows in this tile, in any piece
    const float o_scale = !kWeighted ? 1.0f : w_ref == -INFINITY ? 0.0f : exp2_approx(w_ref - m - kLift);  // O to the units of l
    // Rolled loops: each runs once a segment, and the time of straight code would be that of fetching it.
    const int64_t out_row = ((g.s.first + tiles.tok0(t) + tok) * a.hq + g.h * a.group + head) * static_cast<int64_t>(a.dim);
    if (g.j0 == 0 && g.j1 == g.nt) {
      const float inv = l == 0.0f ? 0.0f : o_scale / l;
      T* const out = static_cast<T*>(a.out) + out_row;
      const bool wide = a.dim % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
#pragma unroll 1
      for (int c = 0; c < a.dim; c += 16) {
        uint32_t o[16], r[8];
        tmem_ld16(tO + c, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = Storage<T>::pack2(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
        if (!valid) continue;
        if (wide) {
          store32(out + c, r);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // head_dim is even, out 4-byte aligned
            if (c + 2 * i < a.dim) *reinterpret_cast<uint32_t*>(out + c + 2 * i) = r[i];
          }
        }
      }
      continue;
    }
    const int run0 = plan.run_of(g.first), run1 = plan.run_of(g.first + g.nt - 1), run = static_cast<int>(blockIdx.x);
    float* const mine = piece_at<DP>(a, 2 * static_cast<int64_t>(run) + (run == run0 ? 1 : 0), t);
    if (active) {
#pragma unroll 1
      for (int c = 0; c < DP; c += 16) {
        uint32_t o[16];
        tmem_ld16(tO + c, o);
        tmem_wait_ld();
        if constexpr (kWeighted) {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * o_scale);
        }
        if (valid) {
          const uint32_t lo[8] = {o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7]}, hi[8] = {o[8], o[9], o[10], o[11], o[12], o[13], o[14], o[15]};
          store32(mine + row * DP + c, lo);
          store32(mine + row * DP + c + 8, hi);
        }
      }
    }
    __stcg(mine + DP * 128 + row, m);
    __stcg(mine + (DP + 1) * 128 + row, l);
    __syncwarp();
    uint32_t* const counter = a.counters + run0 * kCountersPerCta + t * 4 + warp;
    uint32_t before = 0;
    if (lane == 0) before = atom_add_acq_rel_gpu(counter, 1u);
    before = __shfl_sync(0xffffffffu, before, 0);
    if (before != static_cast<uint32_t>(run1 - run0)) continue;
    // Last: the pieces' sum, weighted by their maxima, in their order.
    fence_acq_rel_gpu();
    __syncwarp();
    const int pieces = run1 - run0 + 1, row0 = warp * 32;
    auto piece = [&](int k) { return piece_at<DP>(a, 2 * static_cast<int64_t>(run0 + k) + (k == 0 ? 1 : 0), t); };
    float top = -INFINITY, total = 0.0f;  // a lane a row
#pragma unroll 4
    for (int k = 0; k < pieces; ++k) {
      const float* const pc = piece(k) + DP * 128 + row;
      const float pm = __ldcg(pc), pl = __ldcg(pc + 128);
      if (pl == 0.0f) continue;  // a piece without a sum has no O
      const float higher = max3(top, top, pm);
      total = total * exp2_approx(top - higher) + pl * exp2_approx(pm - higher);
      top = higher;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    constexpr int kCols = DP / 32;  // a lane's columns of a row
    using Vf = Vec<float, kCols < 4 ? kCols : 4>;
    const int held = __popc(__ballot_sync(0xffffffffu, valid));  // the first rows
    constexpr int kAtOnce = kCols == 8 ? 2 : 4;  // rows of two pieces in flight, as many as the registers hold
#pragma unroll 1
    for (int r0 = 0; r0 < held; r0 += kAtOnce) {
      float acc[kAtOnce][kCols];
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r) {
#pragma unroll
        for (int i = 0; i < kCols; ++i) acc[r][i] = 0.0f;
      }
#pragma unroll 1
      for (int k0 = 0; k0 < pieces; k0 += 2) {
        Vf x[kAtOnce][2][kCols < 4 ? 1 : kCols / 4];
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float* const from = piece(min(k0 + k, pieces - 1)) + (row0 + min(31, r0 + r)) * DP + lane * kCols;
#pragma unroll
            for (int i = 0; i < kCols; i += sizeof(Vf) / 4) x[r][k][i * 4 / sizeof(Vf)] = load_cg<Vf>(from + i);
          }
        }
        // The first lanes weigh the rows' two pieces.
        const int rr = min(31, r0 + (lane >> 1 & (kAtOnce - 1))), kk = k0 + (lane & 1);
        const float row_top = __shfl_sync(0xffffffffu, top, rr);
        float f = 0.0f;
        if (kk < pieces && lane < 2 * kAtOnce) {
          const float* const pc = piece(kk) + DP * 128 + row0 + rr;
          const float pm = __ldcg(pc), pl = __ldcg(pc + 128);
          f = pl == 0.0f ? 0.0f : exp2_approx(pm - row_top);
        }
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float fr = __shfl_sync(0xffffffffu, f, 2 * r + k);
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
              const float v = x[r][k][i * 4 / sizeof(Vf)].v[i % (sizeof(Vf) / 4)];
              acc[r][i] = fr == 0.0f ? acc[r][i] : fmaf(fr, v, acc[r][i]);
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r) {
        const int from = min(31, r0 + r);
        const float row_inv = __shfl_sync(0xffffffffu, inv, from);
        const int64_t at = __shfl_sync(0xffffffffu, out_row, from) + lane * kCols;
        if (r0 + r < held && lane * kCols < a.dim) {
#pragma unroll
          for (int i = 0; i < kCols; i += 2) {
            *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at + i) = Storage<T>::pack2(acc[r][i] * row_inv, acc[r][i + 1] * row_inv);
          }
        }
      }
    }
    if (lane == 0) __stcg(counter, 0u);
  }
}

template <typename T, int DP, int CODE>
__global__ void __launch_bounds__(Layout<DP, CODE>::kThreads, 1) tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                                                           const __grid_constant__ CUtensorMap mv, const __grid_constant__ Args a) {
  using L = Layout<DP, CODE>;
  extern __shared__ uint8_t smem_raw[];
  Smem sm;
  sm.ptr = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  sm.base = smem_u32(sm.ptr);
  sm.bars = sm.base + L::kBars;
  sm.words = reinterpret_cast<volatile int*>(sm.ptr + L::kWords);
  sm.status = a.status;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < L::kBarCount; ++i) {
      // P comes from a tile's four warps; a stage is filled by TMA or the four widening warps and given back by both
      // tiles' products and by the warp on V, which follows every one.
      int count = 1;
      if (i >= kPReady0 && i <= kPRest1) count = 4;
      if (i >= L::kFull && i < L::kEmpty) count = L::kCoded ? 4 : 1;
      if (i >= L::kEmpty && i < L::kRawFull) count = 3;
      if (i >= L::kRawEmpty) count = 4;
      mbar_init(sm.bar(i), count);
    }
    fence_barrier_init();
    sm.words[kDead] = 0;
    tma_prefetch_descriptor(&mq);
    tma_prefetch_descriptor(&mk);
    tma_prefetch_descriptor(&mv);
  }
  wait_prior_grid();
  allow_next_grid();
  __syncwarp();
  if (warp == kFixWarp) {  // not before the previous grid has ended: a CTA of it could wait for these columns
    tmem_alloc(sm.base + L::kWords + 4 * kTmem, 512);
    tmem_relinquish();
  }

  // The sequences' units, a run of sequences a thread; every CTA's run of units, and the sequence where this one's begins.
  const int per = (a.batch + L::kThreads - 1) / L::kThreads;
  const int lo = min(a.batch, tid * per), hi = min(a.batch, lo + per);
  int64_t mine = 0;
  for (int b = lo; b < hi; ++b) {
    const Seq s = read_seq(a, b, blockIdx.x == 0);
    mine += s.n > 0 ? head_units(a, s) * a.hkv : 0;
  }
  int64_t inc = mine;
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, k);
    if (lane >= k) inc += y;
  }
  volatile int64_t* const scan = reinterpret_cast<volatile int64_t*>(sm.ptr + L::kWords + 4 * ((kScan + 1) / 2 * 2));
  if (lane == 31) scan[warp] = inc;
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  int64_t before = inc - mine;
  Plan plan{0, 0};
  for (int k = 0; k < L::kThreads / 32; ++k) {
    if (k < warp) before += scan[k];
    plan.total += scan[k];
  }
  plan.runs = static_cast<int>(min(static_cast<int64_t>(gridDim.x), plan.total));
  const bool busy = static_cast<int>(blockIdx.x) < plan.runs;
  int64_t u0 = 0, u1 = 0;
  if (busy) {
    u0 = plan.begin(blockIdx.x);
    u1 = plan.begin(blockIdx.x + 1);
    if (u0 >= before && u0 < before + mine) {
      int64_t off = u0 - before;
      for (int b = lo; b < hi; ++b) {
        const Seq s = read_seq(a, b, false);
        const int64_t n = s.n > 0 ? head_units(a, s) * a.hkv : 0;
        if (off < n) {
          sm.words[kStartSeq] = b;
          sm.words[kStartFirst] = static_cast<int>(s.first);
          sm.words[kStartN] = s.n;
          sm.words[kStartLen] = s.len;
          sm.words[kStartLo] = static_cast<int>(off & 0xffffffff);
          sm.words[kStartHi] = static_cast<int>(off >> 32);
          break;
        }
        off -= n;
      }
    }
  }
  __syncthreads();
  if (busy && warp == 0) find_start(a, sm, lane);
  __syncthreads();
  const uint32_t tmem = static_cast<uint32_t>(sm.words[kTmem]);
  if (busy) {
    Walk w;
    w.init(a, sm, u0, u1);
    if (warp < 8) {
      more_registers<L::kSoftmaxRegs>();
      softmax_role<T, DP, CODE>(a, sm, w, plan, warp >> 2, warp & 3, lane, tmem);
    } else {
      fewer_registers<L::kOtherRegs>();
      if (warp == kLoadWarp) {
        load_role<T, DP, CODE>(a, sm, w, lane, &mq, &mk, &mv);
      } else if (warp < kFixWarp) {
        mma_role<T, DP, CODE>(a, sm, w, warp - kMmaWarp, tmem);
      } else if (warp < kWidenWarp) {
        fix_role<T, DP, CODE>(a, sm, w, lane);
      } else if constexpr (L::kCoded) {
        widen_role<T, DP, CODE>(a, sm, w, tid - kWidenWarp * 32);
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == kFixWarp) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

// ----------------------------------------------------------------- host

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                            const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode encoder() {
  static Encode fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) == cudaSuccess &&
        found == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<Encode>(p);
    }
  });
  return fn;
}

// `bytes` between two entries of a dimension; one of one entry may have any.
cuuint64_t stride_bytes(int64_t elements, int64_t extent, int size) { return extent == 1 ? 16 : static_cast<cuuint64_t>(elements) * size; }

template <typename T, int DP, int CODE>
cudaError_t launch(const Args& a, int sms, cudaStream_t st) {
  using L = Layout<DP, CODE>;
  const Encode enc = encoder();
  if (!enc) return cudaErrorNotSupported;
  const auto type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap mq, mk, mv;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(a.hq), static_cast<cuuint64_t>(a.tokens)};
    const cuuint64_t strides[2] = {stride_bytes(a.dim, a.hq, 2), stride_bytes(a.q_stride, a.tokens, 2)};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(a.tile_tokens)};
    if (enc(&mq, type, 3, const_cast<void*>(a.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
      return cudaErrorInvalidValue;
    }
  }
  for (int i = 0; i < 2; ++i) {
    void* const base = const_cast<void*>(i ? a.v : a.k);
    constexpr int size = L::kCoded ? 1 : 2;
    CUtensorMap* const map = i ? &mv : &mk;
    CUresult r;
    if (a.merged) {
      const cuuint64_t token = stride_bytes(a.token_stride, 0, size);
      const cuuint64_t dims[4] = {64, 8, static_cast<cuuint64_t>(a.head_halves ? a.hkv * L::kHalves : L::kHalves),
                                  static_cast<cuuint64_t>(a.total_groups)};
      const cuuint64_t strides[3] = {token, 128, 8 * token};
      const cuuint32_t box[4] = {64, 8, L::kHalves, static_cast<cuuint32_t>(a.box_rows / 8)};
      r = enc(map, type, 4, base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    } else {
      const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(a.hkv), static_cast<cuuint64_t>(a.page_size),
                                  static_cast<cuuint64_t>(a.num_pages)};
      const cuuint64_t strides[3] = {stride_bytes(a.head_stride, a.hkv, size), stride_bytes(a.token_stride, a.page_size, size),
                                     stride_bytes(a.page_stride, a.num_pages, size)};
      const cuuint32_t box[4] = {L::kCoded ? DP : 64, 1, static_cast<cuuint32_t>(a.box_rows), 1};
      r = enc(map, L::kCoded ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type, 4, base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
              L::kCoded ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    }
    if (r != CUDA_SUCCESS) return cudaErrorInvalidValue;
  }
  const cudaError_t e = cudaFuncSetAttribute(tc_kernel<T, DP, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(true, tc_kernel<T, DP, CODE>, dim3(sms), dim3(L::kThreads), L::kBytes, st, mq, mk, mv, a);
}

template <typename T, int CODE>
cudaError_t launch_dim(const Args& a, int sms, cudaStream_t st) {
  return a.dim <= 64 ? launch<T, 64, CODE>(a, sms, st) : a.dim <= 128 ? launch<T, 128, CODE>(a, sms, st) : launch<T, 256, CODE>(a, sms, st);
}

template <typename T>
cudaError_t launch_for(const Args& a, int code_type, int sms, cudaStream_t st) {
  if (code_type == KL_CODE_E4M3) return launch_dim<T, KL_CODE_E4M3>(a, sms, st);
  if (code_type == KL_CODE_INT8) return launch_dim<T, KL_CODE_INT8>(a, sms, st);
  return launch_dim<T, KL_CODE_NONE>(a, sms, st);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace tc

using namespace tc;

// A box: tokens of one page within 128, a multiple of 8.
static int box_rows_of(int page_size) {
  int r = page_size & -page_size;
  return std::min(r, kBN);
}

// One TMA box for both halves of a row, where head_dim is whole halves and the strides let a head and a page be found
// by halves and groups of 8 tokens; else a box a half. A box takes its warp about 90 cycles to issue, and with pages of
// 16 tokens 32 of them a unit took longer than the unit's products.
static void place_tiles(Args& a, int code_type) {
  const int halves = a.dim <= 64 ? 1 : a.dim <= 128 ? 2 : 4;
  a.group_bytes = 1024;
  a.half_bytes = 128 * 128;
  if (code_type != KL_CODE_NONE || a.dim != 64 * halves) return;
  const int64_t group = 8 * a.token_stride;
  const int64_t page = a.num_pages == 1 ? 0 : a.page_stride, head = a.hkv == 1 ? 0 : a.head_stride;
  if (group <= 0 || page % group != 0) return;
  const bool in_row = head == 64 * halves;  // heads of a token side by side
  if (!in_row && head % group != 0) return;
  const int64_t total = (a.num_pages - 1) * (page / group) + (in_row ? 0 : (a.hkv - 1) * (head / group)) + a.page_size / 8;
  if (total >= INT_MAX) return;
  a.merged = 1;
  a.head_halves = in_row ? halves : 0;
  a.head_groups = in_row ? 0 : static_cast<int>(head / group);
  a.page_groups = static_cast<int>(page / group);
  a.total_groups = static_cast<int>(total);
  a.group_bytes = halves * 1024;
  a.half_bytes = 1024;
}

bool tc_fits(const Args& a, int dtype, int code_type) {
  if (dtype == KL_FLOAT32) return false;
  const int unit = code_type == KL_CODE_NONE ? 8 : 16;  // elements of a cache in 16 bytes
  if (a.dim % 8 != 0 || a.dim % unit != 0 || a.dim > 256 || a.group > 128 || a.page_size % 8 != 0 || !(a.scale_log2 > 0.0f)) return false;
  const auto stride_ok = [](int64_t stride, int64_t extent, int u) {
    return extent == 1 || (stride > 0 && stride % u == 0 && stride < (int64_t(1) << 35));
  };
  return aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && (reinterpret_cast<uintptr_t>(a.out) & 3) == 0 &&
         stride_ok(a.q_stride, a.tokens, 8) && stride_ok(a.head_stride, a.hkv, unit) && stride_ok(a.token_stride, a.page_size, unit) &&
         stride_ok(a.page_stride, a.num_pages, unit) && a.num_pages < INT_MAX;
}

size_t tc_partial_bytes(int head_dim, int sms) {
  const size_t dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  return static_cast<size_t>(sms) * 2 * tiles_of(static_cast<int>(dp)) * (dp + 2) * 128 * sizeof(float);
}

size_t tc_sync_bytes(int sms) { return 256 + static_cast<size_t>(sms) * kCountersPerCta * sizeof(uint32_t); }

cudaError_t launch_tc(Args a, int dtype, int code_type, int sms, cudaStream_t st) {
  a.tile_tokens = 128 / a.group;
  a.block_tokens = (a.dim > 128 ? 1 : 2) * a.tile_tokens;
  a.box_rows = box_rows_of(a.page_size);
  while ((1 << a.box_shift) < a.box_rows) ++a.box_shift;
  place_tiles(a, code_type);
  if (dtype == KL_FLOAT16) return launch_for<__half>(a, code_type, sms, st);
  return launch_for<__nv_bfloat16>(a, code_type, sms, st);
}

}  // namespace chunk_attention
}  // namespace klb
