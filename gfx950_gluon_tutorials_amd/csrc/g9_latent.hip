// Attention over a paged cache of latents (g9_latent_fwd, include/gfx950_fmha.h):
// a token's row holds one latent of 512 values, which is every head's value and the
// larger part of its key, and a rotated key of 64 that the heads share too.
//
// All heads read the same row of 1152 bytes, for 2 (576 + 512) flops each: with 16
// heads the cache's bytes bound the call, with 128 (242 flops a byte) they still
// do by a little, if the products come near the matrix unit's rate.  So a row of the cache
// should reach a CU once for all its heads.
//
// The work is the line of g9_line.hpp, cut into one part per CU.  A workgroup has a block
// of RB = 1, 2 or 4 times 32 query rows and is four waves, one per SIMD with the whole
// register file.  Tiles of 32 keys go through four stages of LDS (147 KB), filled by
// LDS-DMA.  Per tile
//   S^T = K Q^T    by rows: wave w has the rows 32 w .. (their queries are 144 registers a
//                  lane), 36 MFMAs 32x32x16;
//   softmax        of its rows; the weights P go to LDS (16 bit, as the product takes them;
//                  fp32 products have a sixteenth of the rate);
//   O^T += V^T P^T by values: wave w has the values 128 w .. of all rows (64 RB accumulation
//                  registers a lane), 8 RB MFMAs.  V is the row's first 512 values, read
//                  by transposing LDS reads, each once for the workgroup.
// in the register layouts that g9_fmha.hip describes.  (All 512 values of a wave's own
// rows take no exchange, but every wave then reads all of V from LDS.)  A step has the scores
// of tile j + 1 and the values of tile j: the scores' products, which wait for LDS when alone,
// go in turn with some of the values', the softmax and the DMAs of tile j + 3 between the rest.
// A row's maximum moves only where a tile passes it by more than 8 (log2 units); then its
// factor goes through LDS, too.
//
// Measured (us; kernel and join under the profiler, and a call among others; inputs partly in
// the last-level cache): 64 requests of 100 to 8192 tokens (88 K in all) by 16 heads 34-36 + 8 and
// 36-38: 1.5 a tile, 6.1 TB/s over the loop, but 14 go to finding the part, the first loads and
// the sums' way out; by 128 heads 47-49 + 17 and 58-60, 2.1 a tile (68 MFMAs of 32 cycles are 1.2
// at the clock that they leave), 25 outside the loop, much of them and of the join for the
// 256 KB of sums of a part; 16 trees of 12 nodes by 32 heads 79-81 + 16 and, on several cards,
// 85-95; one request of 700 tokens by 16 heads 11 + 4 and 15.
#include "../../include/gfx950_fmha.h"
#include <utility>

#include "g9_attn_host.hpp"
#include "g9_line.hpp"

namespace g9 {
namespace latent {

using namespace fa;

constexpr int kRank = 512, kRow = 576;  // values of a latent, of a row
constexpr int kRowBytes = kRow * 2;
constexpr int kKeys = 32;               // of a tile
constexpr int kTile = kKeys * kRowBytes;
constexpr int kQk = kRow / 16;          // steps of 16 of the scores' product
constexpr int kPv = 4;                  // blocks of 32 values of a wave
constexpr int kAhead = 3;               // steps asked for ahead
// LDS: the stages, P of up to 128 rows, factors of the rows, a word a wave that says
// whether there are any, then the rows' maxima and weights at the end.
constexpr int kP = 4 * kTile, kFactors = kP + 8192, kMoved = kFactors + 512, kMl = kMoved + 64, kLds = kMl + 1024;
constexpr float kNone = -__FLT_MAX__;   // the maximum of a row that has read nothing: finite, weights 0
// From here on (log2 units) a step of fp32 is 2 and more.  A weight's exponent is its score's exact
// product with the scale less the rounded maximum: off by half such a step, and far from 0 for the
// largest score itself.  Then the product is rounded as the maximum is.
constexpr float kLarge = 16777216.f;

struct Params {
  const char* q;
  const char* cache;
  char* o;
  float* lse;                                      // [H][T], or null
  const int* table;
  const int* lengths;
  const int* cu;
  const unsigned long long* mask;                  // or null: a chain
  float* part;                                     // sums of 2 kWgs blocks (part_at), then (m, l) pairs
  Start* start;                                    // [kWgs]: where each part begins
  long long q_t, q_h, o_t, o_h;                    // token / head strides, bytes
  long long c_b;                                   // block stride, bytes
  long long table_stride;
  u32 c_t;                                         // token stride, bytes
  int num_blocks, width, shift, words;
  int B, T, HK, group;                             // HK is 1, group the heads
  float scale_log2;
};

// The sums: 16 blocks of 32 x 32 in all 256 accumulation registers, block N in a[16 N] to
// a[16 N + 15].  They are no variables: the compiler knows the registers as overwritten by each
// statement here and keeps nothing in them (as variables, the sums changed places from loop
// to loop by way of scratch memory; the build checks that no instruction outside assembly names
// one).  The compiler does not look into assembly: the wait states between a product and the
// vector unit's use of its result, or of an operand that the vector unit has just written, are
// `settle` and the s_nop of the statements below (isa_check verifies them).
template <int N>
struct Block;
#define G9_BLOCK(N, LO, HI, ...)                                                                               \
  template <>                                                                                                 \
  struct Block<N> {                                                                                            \
    template <bool BF16>                                                                                       \
    static G9_DEV void product(u32x4 a, u32x4 b) {                                                             \
      if constexpr (BF16)                                                                                      \
        asm volatile("v_mfma_f32_32x32x16_bf16 a[" #LO ":" #HI "], %0, %1, a[" #LO ":" #HI "]"               \
                     : : "v"(a), "v"(b) : __VA_ARGS__);                                                        \
      else                                                                                                     \
        asm volatile("v_mfma_f32_32x32x16_f16 a[" #LO ":" #HI "], %0, %1, a[" #LO ":" #HI "]"                \
                     : : "v"(a), "v"(b) : __VA_ARGS__);                                                        \
    }                                                                                                          \
    template <int E>                                                                                           \
    static G9_DEV void clear() {                                                                               \
      asm volatile("v_accvgpr_write_b32 a%c0, 0" : : "i"(LO + E) : __VA_ARGS__);                              \
    }                                                                                                          \
    template <int E>                                                                                           \
    static G9_DEV void multiply(float f) {                                                                     \
      float x;                                                                                                 \
      asm volatile("v_accvgpr_read_b32 %0, a%c2\n\tv_mul_f32 %0, %0, %1\n\tv_accvgpr_write_b32 a%c2, %0"    \
                   : "=&v"(x) : "v"(f), "i"(LO + E) : __VA_ARGS__);                                           \
    }                                                                                                          \
    template <int E>                                                                                           \
    static G9_DEV float value() {                                                                              \
      float x;                                                                                                 \
      asm volatile("v_accvgpr_read_b32 %0, a%c1" : "=v"(x) : "i"(LO + E) : __VA_ARGS__);                      \
      return x;                                                                                                \
    }                                                                                                          \
  };
G9_BLOCK(0, 0, 15, "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", "a14", "a15")
G9_BLOCK(1, 16, 31, "a16", "a17", "a18", "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", "a27", "a28", "a29", "a30", "a31")
G9_BLOCK(2, 32, 47, "a32", "a33", "a34", "a35", "a36", "a37", "a38", "a39", "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47")
G9_BLOCK(3, 48, 63, "a48", "a49", "a50", "a51", "a52", "a53", "a54", "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63")
G9_BLOCK(4, 64, 79, "a64", "a65", "a66", "a67", "a68", "a69", "a70", "a71", "a72", "a73", "a74", "a75", "a76", "a77", "a78", "a79")
G9_BLOCK(5, 80, 95, "a80", "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", "a91", "a92", "a93", "a94", "a95")
G9_BLOCK(6, 96, 111, "a96", "a97", "a98", "a99", "a100", "a101", "a102", "a103", "a104", "a105", "a106", "a107", "a108", "a109", "a110", "a111")
G9_BLOCK(7, 112, 127, "a112", "a113", "a114", "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", "a124", "a125", "a126", "a127")
G9_BLOCK(8, 128, 143, "a128", "a129", "a130", "a131", "a132", "a133", "a134", "a135", "a136", "a137", "a138", "a139", "a140", "a141", "a142", "a143")
G9_BLOCK(9, 144, 159, "a144", "a145", "a146", "a147", "a148", "a149", "a150", "a151", "a152", "a153", "a154", "a155", "a156", "a157", "a158", "a159")
G9_BLOCK(10, 160, 175, "a160", "a161", "a162", "a163", "a164", "a165", "a166", "a167", "a168", "a169", "a170", "a171", "a172", "a173", "a174", "a175")
G9_BLOCK(11, 176, 191, "a176", "a177", "a178", "a179", "a180", "a181", "a182", "a183", "a184", "a185", "a186", "a187", "a188", "a189", "a190", "a191")
G9_BLOCK(12, 192, 207, "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203", "a204", "a205", "a206", "a207")
G9_BLOCK(13, 208, 223, "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215", "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223")
G9_BLOCK(14, 224, 239, "a224", "a225", "a226", "a227", "a228", "a229", "a230", "a231", "a232", "a233", "a234", "a235", "a236", "a237", "a238", "a239")
G9_BLOCK(15, 240, 255, "a240", "a241", "a242", "a243", "a244", "a245", "a246", "a247", "a248", "a249", "a250", "a251", "a252", "a253", "a254", "a255")
#undef G9_BLOCK

// f<0>(), f<1>(), ..
template <int N, class F>
G9_DEV void each(F f) {
  [&]<int... I>(std::integer_sequence<int, I...>) { (f.template operator()<I>(), ...); }
  (std::make_integer_sequence<int, N>{});
}

template <bool BF16>
G9_DEV void score(f32x16& c, u32x4 a, u32x4 b) {
  if constexpr (BF16)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  else
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
template <bool BF16>
G9_DEV void first_score(f32x16& c, u32x4 a, u32x4 b) {
  if constexpr (BF16)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
  else
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
}
G9_DEV void settle(f32x16& c) { asm volatile("s_nop 7\n\ts_nop 7" : "+v"(c)); }
// The sums' products are done.
G9_DEV void settle() { asm volatile("s_nop 7\n\ts_nop 7"); }

// The lane, worked out where it is used: what follows from it is not held through the loop.
G9_DEV int lane_here() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
}

// RB blocks of 32 rows; a step of the workgroup is a tile.  What a block's beginning and end
// cost, in tiles, is the line's LEAD (us, the cases above with
// 5, 9, 12 places: 128 heads 70, 68.5, 66, trees 99, 97, 98; 16 heads with 5 and 7: 40.5, 41.5;
// 64 rows with 5, 8, 12: 64 requests of 100 to 8192 by 40 heads 87, 85, 85, by 64 90, 87, 86, 256 of
// 100 to 2000 by 64 106, 101, 102).
template <int RB>
using Steps = Line<Params, kKeys, 32 * RB, kWgs, RB == 4 ? 12 : RB == 2 ? 8 : 5>;

// By its bits: comparisons here may take NaN for a number.
G9_DEV bool nothing(float l) { return (__float_as_uint(l) << 1) == 0; }

// One wave: rows 32 wave .. of the block for the scores, values 128 wave .. for the sums.
template <bool BF16, int RB>
struct Wave4 {
  const Params& p;
  int wave;
  u32 lds;             // of the workgroup
  char* smem;
  u32 voff[9];
  u32 ak, av;          // LDS read bases in a tile (K, V)
  u32x4 qf[kQk];
  float m, l;          // of this lane's row
  NodeRow row;
  int keys, whole;     // of the request; keys that every row reads
  u32 bad;             // keys of the tile whose values come next that hold special values
  u32x4 weight[2];     // of the last scores' tile, its softmax's factor and whether that matters
  float factor;
  bool moves;

  G9_DEV explicit Wave4(const Params& pp) : p(pp) {}

  // A tile in LDS: rows of 1152 bytes (72 pieces of 16 bytes, an odd number of 128-byte
  // lines), piece c of row r at place c ^ swz(r).  A K read takes one piece of 16 rows:
  // (r & 1, swz(r)) is different for each, so it touches every bank once.  A
  // transposing V read takes 4 pieces of 4 rows: bit 2 of swz is bit 1 of r.
  static G9_DEV int swz(int r) { return (r >> 1 & 1) << 2 | (r >> 2 & 3); }

  G9_DEV void init(char* sm) {
    const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
    smem = sm;
    lds = (u32)(uintptr_t)to_lds(sm);
    // A wave fetches 8 rows of a tile with nine DMAs: DMA j writes the bytes 1024 j + 16 lane.
#pragma unroll
    for (int j = 0; j < 9; ++j) {
      const int n = 64 * j + lane, r = n / 72;
      voff[j] = (u32)r * p.c_t + 16 * ((n - 72 * r) ^ swz(r + 8 * (wave & 1)));
    }
    ak = lds + col * kRowBytes + 16 * (h ^ swz(col));
    // 16 lanes cover 4 rows and 16 values: lane jj of them row jj / 4, values 4 (jj % 4)
    // of two pieces.
    const int jj = lane & 15, r4 = 4 * h + (jj >> 2);
    av = lds + r4 * kRowBytes + 16 * ((2 * (lane >> 4 & 1) + ((jj & 3) >> 1)) ^ swz(r4)) + 8 * (jj & 1) + 256 * wave;
  }

  // This wave's 8 rows of a tile to come: their descriptor, their place in LDS.
  struct Rows8 {
    rsrc_t r;
    u32 to;
  };
  // Of the tile that begins with key k0, of `all` keys (rows behind them read as zeros), on
  // page pg, into stage `stage`.  A 16-row piece never crosses a page.
  G9_DEV Rows8 aim(int stage, int k0, int all, int pg) const {
    const int k = k0 + 8 * wave, off = k & ((1 << p.shift) - 1);
    const bool in = (u32)pg < (u32)p.num_blocks;
    const int rows = in ? min(max(all - k, 0), 8) : 0;
    const char* const base = p.cache + (long long)(in ? pg : 0) * p.c_b + (unsigned long long)(u32)off * p.c_t;
    return {make_rsrc(uniform(base), uniform(extent(rows, p.c_t, kRowBytes))),
            (u32)uniform((int)(lds + stage * kTile + wave * 8 * kRowBytes))};
  }
  template <int J>
  G9_DEV void fetch(const Rows8& x) const {
    dma16_fresh(x.r, x.to + 1024 * J, voff[J], 0);
  }
  template <int J = 0>
  G9_DEV void fetch_all(const Rows8& x) const {
    if constexpr (J < 9) {
      fetch<J>(x);
      fetch_all<J + 1>(x);
    }
  }

  G9_DEV void load_q(const char* qrow) {
    const int h = lane_here() >> 5;
#pragma unroll
    for (int s = 0; s < kQk; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qrow + (16 * s + 8 * h) * 2);
  }
  G9_DEV void clear() {
    m = kNone, l = 0.f;
    each<RB * kPv>([&]<int B>() { each<16>([&]<int E>() { Block<B>::template clear<E>(); }); });
    asm volatile("s_nop 1");
  }

  // The products of tile j's values (VALUES; P in LDS, the tile in stage `vstage`) and of tile
  // j + 1's scores (SCORES; from key k0 on, stage `kstage`).  The scores come first, in turn
  // with the values' products that their softmax does not need behind them: alone, they would
  // wait for LDS (each wave reads the whole tile for them).  The softmax is cut into pieces of
  // about the 32 cycles that a product takes and goes between the other products.  So do the
  // DMAs of `next`: all at once, they would hold the wave until memory has taken them.  TAIL:
  // tiles that not every row may read whole.
  template <bool SCORES, bool VALUES, bool TAIL>
  G9_DEV void products(int k0, int kstage, int vstage, const Rows8& next) {
    constexpr int kK = SCORES ? kQk : 0, kV = VALUES ? 2 * kPv * RB : 0, kAll = kK + kV;
    constexpr int kDepth = 4;  // K fragments read ahead (the compiler takes assembly for instructions
                               // without a latency, and would read each just before)
    const u32 ks = ak + kstage * kTile, vs = av + vstage * kTile;
    const u32 kb[4] = {ks, ks ^ 32, ks ^ 64, ks ^ 96}, vb[4] = {vs, vs ^ 64, vs ^ 32, vs ^ 96};
    const u32 pb = lds + kP + 16 * (u32)lane_here();
    const auto k_at = [&](int s) { return *(const G9_LDS u32x4*)(uintptr_t)(kb[s & 3] + 128 * (s >> 2)); };
    // Fragment i: block i % 4 of the values, 16 of the keys.
    const auto v_at = [&](int i) {
      const int at = 16 * kRowBytes * (i / kPv) + 128 * (i % kPv >> 1);
      const u32x2 lo = tr_read(vb[i & 1] + at), hi = tr_read(vb[2 + (i & 1)] + at + 8 * kRowBytes);
      return u32x4{lo.x, lo.y, hi.x, hi.y};
    };
    const auto p_at = [&](int rb, int t) { return *(const G9_LDS u32x4*)(uintptr_t)(pb + 1024 * (2 * rb + t)); };
    const u32 out = VALUES && TAIL ? bad >> (4 * (lane_here() >> 5)) : 0;  // of this lane's keys
    u32x4 f[kDepth], v[2], pf[RB];
    f32x16 sc;
    if constexpr (VALUES) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) pf[rb] = p_at(rb, 0);
      v[0] = v_at(0), v[1] = v_at(1);
    }
    if constexpr (SCORES) {
#pragma unroll
      for (int s = 0; s < kDepth; ++s) f[s] = k_at(s);
    }
    // DMA J behind product (2 J + 1) / 18 of all.
    const auto slot = [&]<int S>() {
      constexpr int J = (2 * S + 1) * 9 / (2 * kAll), K = (2 * S + 3) * 9 / (2 * kAll);
      static_assert(K - J <= 2);
      if constexpr (J != K && J < 9) fetch<J>(next);
      if constexpr (K == J + 2 && K <= 9) fetch<J + 1>(next);
    };
    const auto value = [&]<int I>() {
      constexpr int kFrag = I / RB, kBlock = I % RB, kTime = kFrag / kPv;
      u32x4& x = v[kFrag & 1];
      if constexpr (TAIL && kBlock == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u32 two = out >> (16 * kTime + 8 * (e / 2) + 2 * (e % 2));
          x[e] &= (two & 1 ? 0 : 0xffffu) | (two & 2 ? 0 : 0xffff0000u);
        }
        asm volatile("s_nop 1" : "+v"(x));
      }
      Block<kBlock * kPv + kFrag % kPv>::template product<BF16>(x, pf[kBlock]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kFrag == kPv - 1) pf[kBlock] = p_at(kBlock, 1);
      if constexpr (kBlock == RB - 1 && kFrag + 2 < 2 * kPv) x = v_at(kFrag + 2);
    };
    // The softmax: kPieces pieces behind product kLast + 2.
    constexpr int kPieces = 20, kMix = SCORES && kV > kPieces + 2 ? kV - kPieces - 2 : 0;
    constexpr int kLast = kK + kMix - 1;  // the last score's product, at the latest
    constexpr int kSlots = kAll - kLast - 3, kEach = kSlots > 0 ? (kPieces + kSlots - 1) / kSlots : kPieces;
    Soft<TAIL> soft{k0, kstage, p.scale_log2};
    const auto pieces = [&]<int FIRST, int N>() {
      each<N>([&]<int I>() {
        if constexpr (FIRST + I < kPieces) piece<TAIL, FIRST + I>(soft, sc);
      });
    };
    const auto step = [&]<int S>(auto self) {
      // Product S of all.
      if constexpr (S < kAll) {
        constexpr int kBefore = SCORES ? (S <= kLast ? S * kK / (kLast + 1) : kK) : 0;
        constexpr int kBehind = SCORES ? (S < kLast ? (S + 1) * kK / (kLast + 1) : kK) : 0;
        if constexpr (kBehind > kBefore) {
          if constexpr (kBefore == 0)
            first_score<BF16>(sc, f[0], qf[0]);
          else
            score<BF16>(sc, f[kBefore % kDepth], qf[kBefore]);
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (kBefore + kDepth < kK) f[kBefore % kDepth] = k_at(kBefore + kDepth);
        } else {
          value.template operator()<S - kBefore>();
        }
        slot.template operator()<S>();
        if constexpr (SCORES && S > kLast + 2) pieces.template operator()<(S - kLast - 3) * kEach, kEach>();
        self.template operator()<S + 1>(self);
      }
    };
    step.template operator()<0>(step);
    if constexpr (SCORES) pieces.template operator()<(kSlots > 0 ? kSlots * kEach : 0), kPieces>();
    if constexpr (SCORES && TAIL) bad = soft.bad;
  }

  template <bool TAIL>
  struct Soft {
    int k0, stage;
    float scale;  // what is left of it to multiply the scores by
    u32 bad = 0;
    float top = 0.f, sum[2] = {0.f, 0.f};
  };
  // Piece N of the softmax: the maximum of the scores, the weights one by one.
  template <bool TAIL, int N>
  G9_DEV void piece(Soft<TAIL>& x, f32x16& sc) {
    if constexpr (N == 0) {
      settle(sc);
      if constexpr (TAIL) {
        x.bad = x.k0 + kKeys > whole ? special(x.stage) : 0;
        const int h = lane_here() >> 5;
        const u32 reads = (u32)node_reads(p, row, x.k0, keys);
        u32 quiet;  // a NaN that the compiler, told not to mind them, does not see
        asm("v_mov_b32 %0, 0x7fc00000" : "=v"(quiet));
        const u32 bits = reads >> (4 * h), nan = (reads & x.bad) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = 8 * (i / 4) + i % 4;
          const float y = __uint_as_float(nan >> key & 1 ? quiet : __float_as_uint(sc[i]));
          sc[i] = bits >> key & 1 ? y : -__builtin_inff();
        }
      }
      x.top = sc[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) x.top = __builtin_fmaxf(x.top, sc[i]);
    } else if constexpr (N == 1) {
#pragma unroll
      for (int i = 8; i < 16; ++i) x.top = __builtin_fmaxf(x.top, sc[i]);
      x.top = xhalf(x.top, [](float a, float b) { return __builtin_fmaxf(a, b); }) * p.scale_log2;
    } else if constexpr (N == 2) {
      const bool up = x.top - m > kLazyThreshold;
      factor = 1.f, moves = false;
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(up) != 0, 0)) {
        const float m_new = up ? x.top : m;
        factor = __builtin_amdgcn_exp2f(m - m_new);
        // A row's first tile moves its maximum, but not its sums, which are zeros.
        moves = __builtin_amdgcn_ballot_w64(up && (m > kNone || !nothing(l))) != 0;
        m = m_new;
        l *= factor;
      }
      const bool large = __builtin_fabsf(m) >= kLarge;
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(large) != 0, 0)) {
        // The other rows' products are by 1: their weights stay those of their own scores.
        const float by = large ? p.scale_log2 : 1.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] *= by;
        x.scale = large ? 1.f : p.scale_log2;
      }
    } else if constexpr (N < 19) {
      // Weight N - 3, and what follows from those before it.
      constexpr int E = N - 3;
      sc[E] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[E], x.scale, -m));
      if constexpr (E > 0) x.sum[(E - 1) % 2] += sc[E - 1];
      if constexpr (E > 1 && E % 2 == 0) weight[(E - 2) / 8][(E - 2) % 8 / 2] = pack2<BF16>(sc[E - 2], sc[E - 1]);
    } else {
      weight[1][3] = pack2<BF16>(sc[14], sc[15]);
      l += x.sum[0] + (x.sum[1] + sc[15]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  // The weights to LDS behind a barrier (every wave has read the last tile's), with the
  // factors of the rows whose maximum moved.
  G9_DEV void publish() {
    barrier();
    if (wave < RB) {
      const int lane = lane_here();
      G9_LDS u32x4* const to = (G9_LDS u32x4*)(uintptr_t)(lds + kP + 2048 * wave + 16 * lane);
      to[0] = weight[0], to[64] = weight[1];
      *(G9_LDS float*)(uintptr_t)(lds + kFactors + 128 * wave + 4 * (lane & 31)) = factor;
      *(G9_LDS u32*)(uintptr_t)(lds + kMoved + 4 * wave) = moves;
    }
    waitcnt<63, 0>();
  }

  // Whether a row's maximum moved with the last weights.
  G9_DEV bool moved() const {
    const u32x4 x = *(const G9_LDS u32x4*)(uintptr_t)(lds + kMoved);
    const u32 any = RB == 1 ? x.x : RB == 2 ? x.x | x.y : x.x | x.y | x.z | x.w;
    return __builtin_amdgcn_readfirstlane((int)any) != 0;
  }
  // Then all rows' sums are multiplied by their factors before the weights join them.
  G9_DEV void rescale() {
    const u32 at = lds + kFactors + 4 * (lane_here() & 31);
    settle();
    each<RB>([&]<int R>() {
      const float factor = *(const G9_LDS float*)(uintptr_t)(at + 128 * R);
      each<kPv>([&]<int D>() { each<16>([&]<int E>() { Block<R * kPv + D>::template multiply<E>(factor); }); });
    });
    asm volatile("s_nop 1");
  }

  // The keys of the tile that hold an infinite or NaN latent.  A weight of 0 would not
  // keep such a value out of a row that does not read its key: where not every row
  // reads every key, these keys' values are left out of the product, and the rows that do
  // read one get a score of NaN (the latent is the key too: its product with the
  // query would be infinite or NaN).
  G9_DEV u32 special(int stage) const {
    typedef unsigned short h2 __attribute__((ext_vector_type(2)));
    constexpr u32 kExp = BF16 ? 0x7f80u : 0x7c00u;
    h2 top = {0, 0};
    const int lane = lane_here(), h = lane >> 5, col = lane & 31;
    // Half a latent a lane; the order of its pieces so that 16 rows touch every bank once.
    const u32 at = lds + stage * kTile + col * kRowBytes + 512 * h + 16 * (col >> 1 & 7);
#pragma unroll 8
    for (int j = 0; j < 32; ++j) {
      const u32x4 x = *(const G9_LDS u32x4*)(uintptr_t)((at ^ (16 * (j & 7))) + 128 * (j >> 3));
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(h2, x[e] & 0x7fff7fffu));
    }
    const unsigned long long who = __builtin_amdgcn_ballot_w64(top.x >= kExp || top.y >= kExp);
    return (u32)who | (u32)(who >> 32);
  }
};

// Sums in the workspace: [slot][32 rows][64 groups of 8 values][lane][4], as the products
// leave them, a lane being a row and half of the 8 values: whole lines, written and read.
template <int RB>
G9_DEV size_t part_at(size_t slot, int rb, int q) {
  return (((slot * RB + rb) * 64 + q) * 64) * 4;
}
template <int RB>
G9_DEV size_t ml_at(size_t slot, int row) {
  return (size_t)2 * kWgs * 32 * RB * kRank + (slot * 32 * RB + row) * 2;
}
// Where a lane's row goes: row `in` of the block.
struct Out {
  char* o;
  float* lse;
};
template <class P>
G9_DEV Out out_of(const P& p, int q0, int row, int node) {
  const int hq = row - node * p.group;
  const long long tok = q0 + node;
  return {p.o + tok * p.o_t + hq * p.o_h, p.lse ? p.lse + (long long)hq * p.T + tok : nullptr};
}
template <bool BF16>
G9_DEV u32x2 scaled(f32x4 x, float inv) {
  return u32x2{pack2<BF16>(x[0] * inv, x[1] * inv), pack2<BF16>(x[2] * inv, x[3] * inv)};
}
G9_DEV float lse_of(float m, float l) { return nothing(l) ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2; }

// A block's results, or its sums to slot `slot` of the workspace: the rows' maxima and weights
// go through LDS from the waves that have them.  Branches of lanes are not nested: nothing
// may come between the ends of two of them.
template <bool BF16, int RB, class L>
G9_DEV void finish_block(const Params& p, const Place& at, int slot, Wave4<BF16, RB>& w) {
  const int lane = lane_here(), h = lane >> 5, col = lane & 31;
  const float l = xhalf(w.l, [](float x, float y) { return x + y; });
  waitcnt<0, 15>();  // the DMAs behind the last step
  if (h == 0) *reinterpret_cast<f32x2*>(w.smem + kMl + 256 * w.wave + 8 * col) = f32x2{w.m, l};
  __syncthreads();  // and every wave has read its tiles
  settle();
  each<RB>([&]<int R>() {
    const f32x2 ml = *reinterpret_cast<const f32x2*>(w.smem + kMl + 256 * R + 8 * col);
    // Values 8 I + 4 h .. of this wave's 128.
    const auto quad = [&]<int I>() {
      using B = Block<R * kPv + I / 4>;
      constexpr int kFirst = 4 * (I % 4);
      return f32x4{B::template value<kFirst>(), B::template value<kFirst + 1>(), B::template value<kFirst + 2>(),
                   B::template value<kFirst + 3>()};
    };
    if (slot >= 0) {
      float* const to = p.part + part_at<RB>(slot, R, 16 * w.wave) + 4 * lane;
      each<16>([&]<int I>() { *reinterpret_cast<f32x4*>(to + 256 * I) = quad.template operator()<I>(); });
      if (w.wave == R && h == 0) *reinterpret_cast<f32x2*>(p.part + ml_at<RB>(slot, 32 * R + col)) = ml;
    } else {
      const int row = at.block * L::kBlock + 32 * R + col, node = row_of<L>(p, at, 32 * R + col).node;
      const Out out = out_of(p, at.r.q0, row, max(node, 0));
      const float inv = nothing(ml.y) ? 0.f : 1.f / ml.y;
      if (node >= 0)
        each<16>([&]<int I>() {
          *reinterpret_cast<u32x2*>(out.o + 256 * w.wave + 16 * I + 8 * h) = scaled<BF16>(quad.template operator()<I>(), inv);
        });
      if (w.wave == R && h == 0 && node >= 0 && out.lse) *out.lse = lse_of(ml.x, ml.y);
    }
  });
}

// Joins the blocks that are cut.  A block of n parts has the n - 1 workers whose parts
// begin within it, and with each of them gridDim.y workgroups here, which share its groups
// of 32 rows by 8 values: a wave each where the parts are few, else a workgroup, whose
// waves share the parts.  In the order of the keys: with m the largest of the parts'
// maxima, the sum of 2^(m_i - m) O_i over the sum of 2^(m_i - m) l_i.
constexpr int kJoinWaves = 8, kFewParts = 8, kJoinUnits = 4;
constexpr int kJoinLds = kJoinWaves * 64 * (4 * kJoinUnits + 2);
template <bool BF16, int RB>
G9_DEV void join_parts(const Params& p, float* lds) {
  using L = Steps<RB>;
  const unsigned w = blockIdx.x + 1;
  const Start zero = p.start[0];
  const unsigned long long total = (unsigned long long)zero.total_hi << 32 | zero.total_lo;
  const Start st = p.start[w];  // asked for together with worker 0's
  if (w >= L::workers(total) || st.tile == 0) return;
  const unsigned long long u0 = L::part_begin(w, total) - (unsigned)st.tile;  // the block's first tile
  const unsigned w0 = L::worker_of(u0, total), n = L::worker_of(u0 + st.tiles - 1, total) - w0 + 1;
  const int row0 = st.block * L::kBlock;
  const int rows = (int)min((long long)st.n * p.group - row0, (long long)L::kBlock);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int share = (int)((w - w0 - 1) * gridDim.y + blockIdx.y), shares = (int)((n - 1) * gridDim.y);
  const int units = (rows + 31) / 32 * 64;
  // The worker in whose part the block begins has it in slot 1, the others in slot 0.
  const auto slot_of = [&](unsigned i) { return i ? (size_t)2 * (w0 + i) : (size_t)2 * w0 + 1; };
  const auto store = [&](int u, f32x4 x, float m, float l) {
    const int q = u & 63, row = row0 + 32 * (u >> 6) + (lane & 31), node = row / p.group;
    const Out out = out_of(p, st.q0, row, node);
    *reinterpret_cast<u32x2*>(out.o + 16 * q + 8 * h) = scaled<BF16>(x, nothing(l) ? 0.f : 1.f / l);
    if (q == 0 && h == 0 && out.lse) *out.lse = lse_of(m, l);
  };
  // The sums of U units from u on over the parts k0, k0 + step, .., 16 loads and their maxima
  // and weights asked for together, and what they find scaled to the largest maximum so far.
  const auto sum_parts = [&]<int U>(int u, unsigned k0, unsigned step, f32x4 (&sum)[U], float& m, float& l) {
    constexpr unsigned kAtOnce = 16 / U;
    const int rb = u >> 6, q = u & 63, in = 32 * rb + (lane & 31);
    m = kNone, l = 0.f;
#pragma unroll
    for (int i = 0; i < U; ++i) sum[i] = f32x4{};
    for (unsigned k = k0; k < n; k += kAtOnce * step) {
      f32x4 x[kAtOnce][U];
      f32x2 v[kAtOnce];
#pragma unroll
      for (unsigned e = 0; e < kAtOnce; ++e) {
        const size_t slot = slot_of(min(k + e * step, n - 1));
        v[e] = *reinterpret_cast<const f32x2*>(p.part + ml_at<RB>(slot, in));
        const f32x4* const at = reinterpret_cast<const f32x4*>(p.part + part_at<RB>(slot, rb, q) + 4 * lane);
#pragma unroll
        for (int j = 0; j < U; ++j) x[e][j] = at[64 * j];
      }
      float top = m;
#pragma unroll
      for (unsigned e = 0; e < kAtOnce; ++e)
        if (k + e * step < n) top = __builtin_fmaxf(top, v[e].x);
      const float g = __builtin_amdgcn_exp2f(m - top);
      m = top, l *= g;
#pragma unroll
      for (int j = 0; j < U; ++j) sum[j] *= g;
#pragma unroll
      for (unsigned e = 0; e < kAtOnce; ++e) {
        if (k + e * step >= n) break;
        const float f = __builtin_amdgcn_exp2f(v[e].x - m);
        l += f * v[e].y;
#pragma unroll
        for (int j = 0; j < U; ++j) sum[j] += f * x[e][j];
      }
    }
  };
  if (n <= kFewParts) {
    const auto run = [&]<int U>() {
      for (int u = (share * kJoinWaves + wave) * U; u < units; u += shares * kJoinWaves * U) {
        f32x4 sum[U];
        float m, l;
        sum_parts.template operator()<U>(u, 0, 1, sum, m, l);
        if (32 * (u >> 6) + (lane & 31) < rows)
#pragma unroll
          for (int i = 0; i < U; ++i) store(u + i, sum[i], m, l);
      }
    };
    if (n <= 4)
      run.template operator()<4>();
    else
      run.template operator()<2>();
    return;
  }
  const auto run = [&]<int U>() {
    constexpr int kWords = 4 * U + 2;
    for (int u = share * U; u < units; u += shares * U) {
      f32x4 sum[U];
      float m, l;
      sum_parts.template operator()<U>(u, wave, kJoinWaves, sum, m, l);
      float* const mine = lds + wave * 64 * kWords + lane;  // words 64 apart: a bank a lane
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[64 * (4 * i + e)] = sum[i][e];
      mine[64 * 4 * U] = m, mine[64 * (4 * U + 1)] = l;
      __syncthreads();
      if (wave < U && 32 * (u >> 6) + (lane & 31) < rows) {
        const auto of = [&](int i, int word) { return lds[(i * kWords + word) * 64 + lane]; };
        float m_all = kNone, l_all = 0.f;
#pragma unroll
        for (int i = 0; i < kJoinWaves; ++i) m_all = __builtin_fmaxf(m_all, of(i, 4 * U));
        f32x4 x = {};
#pragma unroll
        for (int i = 0; i < kJoinWaves; ++i) {
          const float f = __builtin_amdgcn_exp2f(of(i, 4 * U) - m_all);
          l_all += f * of(i, 4 * U + 1);
          x += f * f32x4{of(i, 4 * wave), of(i, 4 * wave + 1), of(i, 4 * wave + 2), of(i, 4 * wave + 3)};
        }
        store(u + wave, x, m_all, l_all);
      }
      __syncthreads();
    }
  };
  if (units <= shares)
    run.template operator()<1>();
  else
    run.template operator()<kJoinUnits>();
}

template <bool BF16, int RB>
G9_DEV void fwd(const Params& p, char* smem) {
  using L = Steps<RB>;
  using W = Wave4<BF16, RB>;
  const unsigned worker = my_part();
  Place cur{};
  int left = L::template locate<256>(p, smem, worker, cur);
  W w(p);
  w.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  w.init(smem);
  while (left > 0) {
    const int seg = min(left, cur.r.tiles - cur.tile);
    const bool last = cur.tile + seg == cur.r.tiles, from_start = cur.tile == 0;
    const int first = cur.tile * kKeys;  // the part's first key
    const int in_block = 32 * w.wave + (lane_here() & 31);
    // This wave has rows.  One that has none (with RB 1 and 2 some never do) forms the first
    // row's weights all the same, and no one reads them: the others take as long.
    const bool some = w.wave < RB && cur.block * L::kBlock + 32 * w.wave < cur.r.n * p.group;
    w.row = row_of<L>(p, cur, some ? in_block : 0);
    w.keys = cur.r.keys;
    w.whole = min(cur.r.context, cur.r.keys);
    // The pages of 32 steps' tiles, two 16-row pieces each, are held in the lanes: a load in
    // every step would be waited for in it, as scalar loads are behind the next LDS read.
    const int* const table = p.table + cur.b * p.table_stride;
    const auto pages = [&](int step) {
      const int lane = lane_here(), k = first + (step + (lane >> 1)) * kKeys + 16 * (lane & 1);
      return k < cur.r.keys ? table[k >> p.shift] : -1;
    };
    int held = pages(0);
    __builtin_amdgcn_sched_barrier(0);  // the queries come behind the pages
    const auto rows_of = [&](int step) {
      return w.aim(step & 3, first + step * kKeys, step < seg ? cur.r.keys : 0,
                   __builtin_amdgcn_readlane(held, 2 * (step & 31) + (w.wave >> 1)));
    };
    w.load_q(query_of<L>(p, cur, some ? in_block : 0, w.row.node));
    __builtin_amdgcn_sched_barrier(0);
    w.fetch_all(rows_of(0));
    w.clear();
    waitcnt<0, 0>();  // here: a wait of the compiler's for the queries would be one in every step
    w.fetch_all(rows_of(1));
    barrier();  // tile 0 has landed
    w.template products<true, false, true>(first, 0, 0, rows_of(2));
    w.publish();
    waitcnt<9, 15>();
    barrier();  // tile 1 has landed, P and the factors are there
    // Step j: the values of tile j, the scores and weights of tile j + 1.
    const auto step = [&]<bool TAIL>(int j) {
      if (((j + kAhead) & 31) == 0) {
        held = pages(j + kAhead);
        waitcnt<0, 15>();
      }
      w.template products<true, true, TAIL>(first + (j + 1) * kKeys, (j + 1) & 3, j & 3, rows_of(j + kAhead));
      w.publish();
      waitcnt<9, 15>();
      barrier();  // tile j + 2 has landed, P and the factors are there
    };
    // The steps of tiles that every row reads whole, then the others; the last tile's values.
    // The loops are left to multiply the sums: in them, that code would cost registers.
    const int mid = min((w.whole - first) / kKeys - 1, seg - 1);
    int j = 0;
    for (;;) {
      if (__builtin_expect(w.moved(), 0)) w.rescale();
      if (j < mid) {
        do step.template operator()<false>(j++);
        while (j < mid && !w.moved());
      } else if (j < seg - 1) {
        step.template operator()<true>(j++);
      } else {
        break;
      }
    }
    w.template products<false, true, true>(0, 0, j & 3, rows_of(j + kAhead));
    const int slot = last && from_start ? -1 : (int)(2 * worker + (from_start ? 1 : 0));
    finish_block<BF16, RB, L>(p, cur, slot, w);
    __syncthreads();  // the maxima and weights are read
    left -= seg + L::kLead;
    if (left > 0) cur = L::next_block(p, cur);
  }
}

}  // namespace latent
}  // namespace g9

using namespace g9;
using namespace g9::host;

#define G9_LATENT_KERNEL(NAME, BF16, RB)                                                                           \
  extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void                    \
  g9_latent_##NAME(latent::Params p) {                                                                            \
    __shared__ __attribute__((aligned(1024))) char smem[latent::kLds];                                            \
    latent::fwd<BF16, RB>(p, smem);                                                                               \
  }                                                                                                               \
  extern "C" __global__ __launch_bounds__(64 * latent::kJoinWaves) void g9_latent_join_##NAME(latent::Params p) { \
    __shared__ float lds[latent::kJoinLds];                                                            \
    latent::join_parts<BF16, RB>(p, lds);                                                                         \
  }
G9_LATENT_KERNEL(bf16_q32, true, 1)
G9_LATENT_KERNEL(f16_q32, false, 1)
G9_LATENT_KERNEL(bf16_q64, true, 2)
G9_LATENT_KERNEL(f16_q64, false, 2)
G9_LATENT_KERNEL(bf16_q128, true, 4)
G9_LATENT_KERNEL(f16_q128, false, 4)

namespace {

// Query rows of a block, by the rows (nodes by heads) that a request of the batch
// brings on average: the fewest that hold them, and 128 above (us with 32, 64 and 128 rows; 64
// requests, their lengths spread evenly over 100 to 8192: 265 K tokens, three times the bytes of the
// case above, and each call behind 1 GiB of writes; by 16 heads 123, 125, 133, 32: 136, 139,
// 142, 40: 167, 142, 148, 64: 167, 143, 153, 80: 222, 188, 159, 128: 200, 149, 144; 16 requests
// of 12 nodes by 16 heads 102, 79, 72.  One call behind another: 64 requests by 40 heads 122,
// 85, 97, by 64 126, 87, 99, 16 of 4 nodes by 16 48, 41, 48, 4 of 8000 to 16000 by 64 34, 32, 41.
// But a single request takes the fewer rows: 30000 tokens by 128 heads 44, 44, 56, by 64 31,
// 36, 42, 700 by 64 16, 20, 21).
enum { Q32, Q64, Q128 };
int form_of(int64_t B, int64_t T, int64_t H) {
  const int64_t rows = (T + B - 1) / B * H;
  return rows <= 32 ? Q32 : rows <= 64 ? Q64 : Q128;
}
// Workgroups of the join for each worker: the more, the larger a part (us, the join alone: one
// request by 16 heads with 1 and 2 4.4 and 5.6, 64 requests 6.8 and 6.5; by 128 heads with 2, 4
// and 8 16.8, 15.6 and 14.2, trees 20, 15.3 and 15.8; 64 rows with 1, 2 and 4, whole calls: 64
// requests by 64 heads 87, 87 and 86, 256 of 100 to 2000 102, 101 and 100, 4 of 8000 to 16000 32, 32
// and 35).
constexpr unsigned join_shares(int form) { return 1u << form; }
// The workspace: the sums of 2 x 256 blocks and their (m, l) pairs, then start[].
size_t start_at(int form) { return (size_t)2 * fa::kWgs * (32 << form) * (512 + 2) * 4; }

#define G9_LATENT_FN(WHAT, Q) {reinterpret_cast<const void*>(WHAT##f16_##Q), reinterpret_cast<const void*>(WHAT##bf16_##Q)}
const void* const kRun[3][2] = {G9_LATENT_FN(g9_latent_, q32), G9_LATENT_FN(g9_latent_, q64), G9_LATENT_FN(g9_latent_, q128)};
const void* const kJoin[3][2] = {G9_LATENT_FN(g9_latent_join_, q32), G9_LATENT_FN(g9_latent_join_, q64),
                                 G9_LATENT_FN(g9_latent_join_, q128)};

}  // namespace

extern "C" size_t g9_latent_workspace_size(int64_t B, int64_t T, int64_t H) {
  if (B <= 0 || T <= 0 || H <= 0) return 0;
  return start_at(form_of(B, T, H)) + fa::kWgs * sizeof(fa::Start);
}

extern "C" int g9_latent_fwd(const void* q, const void* cache, void* o, float* lse, const int32_t* block_table,
                             int64_t table_stride, int64_t width, const int32_t* lengths, const int32_t* cu_q,
                             const int64_t* tree_mask, int64_t words, int64_t B, int64_t T, int64_t H,
                             int64_t num_blocks, int64_t block_size, const int64_t* q_strides,
                             const int64_t* cache_strides, const int64_t* o_strides, float sm_scale, int dtype,
                             void* workspace, size_t workspace_bytes, void* stream) {
  using latent::kRank, latent::kRow;
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (B < 0 || B > G9_TREE_MAX_REQUESTS || T < 0 || T > kMaxRows || H <= 0 || H > 65536 || !scale_ok(sm_scale) ||
      num_blocks < 0 || num_blocks > kMaxRows || width < 0 || width > kMaxRows || !block_size_ok(block_size) ||
      width * block_size > (int64_t(1) << 30) || words < 0 || words > 1024 || (tree_mask && words == 0))
    return G9_ERR_SHAPE;
  if (!q_strides || !cache_strides || !o_strides) return G9_ERR_LAYOUT;
  // The step of a single row is never taken.
  const int64_t qs[2] = {T > 1 ? q_strides[0] : 0, H > 1 ? q_strides[1] : 0};
  const int64_t os[2] = {T > 1 ? o_strides[0] : 0, H > 1 ? o_strides[1] : 0};
  const int64_t cs[2] = {num_blocks > 1 ? cache_strides[0] : 0, cache_strides[1]};
  if (!steps(qs, 2) || !steps(cs, 2) || !steps(os, 2)) return G9_ERR_LAYOUT;
  const int64_t size[2] = {T, H};
  if (!apart(size, os, 2, kRank) || (B > 1 && table_stride < width)) return G9_ERR_LAYOUT;
  // A 16-row piece of a page lies within a descriptor's range, its rows apart.
  if (cs[1] < kRow || cs[1] * 2 * 16 >= (int64_t(1) << 31)) return G9_ERR_LAYOUT;
  if (T * H > INT32_MAX) return G9_ERR_SHAPE;
  if (B == 0 || T == 0) return G9_OK;
  if (!q || !o || !lengths || !cu_q || (width && !block_table) || (num_blocks && !cache)) return G9_ERR_LAYOUT;
  if (!aligned16(q) || !aligned16(cache) || !aligned16(o) || ((uintptr_t)lse & 3) || ((uintptr_t)tree_mask & 7))
    return G9_ERR_LAYOUT;
  const int form = form_of(B, T, H);
  if (!workspace || ((uintptr_t)workspace & 31) || workspace_bytes < g9_latent_workspace_size(B, T, H))
    return G9_ERR_WORKSPACE;
  latent::Params p{};
  p.q = static_cast<const char*>(q);
  p.cache = static_cast<const char*>(cache);
  p.o = static_cast<char*>(o);
  p.lse = lse;
  p.table = block_table;
  p.lengths = lengths;
  p.cu = cu_q;
  p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  p.part = static_cast<float*>(workspace);
  p.start = reinterpret_cast<fa::Start*>(static_cast<char*>(workspace) + start_at(form));
  p.q_t = qs[0] * 2, p.q_h = qs[1] * 2, p.o_t = os[0] * 2, p.o_h = os[1] * 2;
  p.c_b = cs[0] * 2, p.c_t = (u32)(cs[1] * 2);
  p.table_stride = table_stride;
  p.num_blocks = (int)num_blocks, p.width = (int)width, p.shift = log2_of(block_size), p.words = (int)words;
  p.B = (int)B, p.T = (int)T, p.HK = 1, p.group = (int)H;
  p.scale_log2 = sm_scale * fa::kLog2e;
  void* args[] = {&p};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int bf16 = dtype == G9_BF16;
  if (hipLaunchKernel(kRun[form][bf16], dim3(fa::kWgs), dim3(256), args, 0, st) != hipSuccess) return G9_ERR_HIP;
  return launched(hipLaunchKernel(kJoin[form][bf16], dim3(fa::kWgs - 1, join_shares(form)),
                                  dim3(64 * latent::kJoinWaves), args, 0, st));
}
