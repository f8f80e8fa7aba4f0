// Attention over the 8-bit cache for many query rows per request and kv head: prompts and chunks of them.
//
// A CTA owns 256 query rows (tokens x heads of one kv head) as two tiles of 128 and walks the keys in tiles of 128,
// in two steps of 64 each.  Its warps:
//   loader       looks up blocks and scales of the next key tile and fetches its levels with TMA
//   converters   levels -> f16 (exact) in the 128-byte swizzled layout of the tensor core's operands; the rows of a
//                tile are keys, 64 values wide, which reads as K-major for Q K^T and as MN-major for P V alike
//   two issuers  one thread per query tile: S = Q K^T and O += P V with tcgen05.mma kind::f16; O in TMEM, S in two
//                buffers of 64 columns per query tile, P as the TMEM operand in the columns that its S had.  The
//                scores of step u + 1 are there before the softmax of step u ends; while one tile's thread waits the
//                other tile's products run.
//   softmax      a warpgroup per query tile, a thread per row: running maximum in the scale of log2, exp2, sums in
//                fp32; O is rescaled only when a maximum has grown by 2^kSlack.
// Few rows over a long cache: several CTAs take shares of an item's keys (launch_of) and a second kernel joins them.
// Key scales multiply the scores of their 16 keys.  Value scales multiply P: a row of O is in units of the largest
// product of a probability and its value scale so far, so that P stays in the range of f16 and keeps its bits whatever
// scales the blocks have that have little part in it; see kPScaleLog2.
// What bounds it, at dim 128 per 256 rows and 128 keys (about 3950 cycles in all), by count: shared memory 3070 cycles
// (levels in and out 512, operands out 512, Q and K into S 1536 at 64 keys a product, V into O 512), exp2 2048 at 16 a
// cycle less the quarter that goes to the FMA pipe, products 2560 (a product of 64 keys takes 49 cycles, not 32).  Of a
// profiled call the tensor pipe was active 0.48, instructions were issued 0.57 and the conversion and exp2 pipe was busy
// 0.37 of the time: no unit is at its end, the chain from scores to P to products goes through all of them in turn.
// Measured at 4095 tokens behind 12289, 32 over 8 heads in bf16: 0.91 to 1.05 ms by card and clock = 920 to 1060 TFLOP/s,
// 0.56 to 0.64 of the measured bf16 rate.  What was measured on the way
// there, in the order of the steps, beside 0.98: scores of 128 keys in one buffer 1.07 ms (the chain softmax, P V, S is
// exposed), one issuer for both tiles 1.44,
// products issued behind `lane == 0` 1.20, levels to registers instead of TMA 1.40, exp2 all on the MUFU 1.01, half of
// them on the FMA pipe 1.08, taking turns in exp2 1.02.  Short prompts pay for the start of a CTA (8300 cycles to the
// first score) and its end (3900): 4 prompts of 256 to 2048 tokens, 32 heads: 140 us = 470 TFLOP/s in f16.
#include "kv8.h"

#include <algorithm>
#include <type_traits>

#include "device_info.h"
#include "kv8_attention.cuh"

namespace disc_b200 {

__device__ int g_kv8_prefill_status = 0;

namespace {

constexpr int kTile = 128;               // query rows of a tile and keys of a tile
constexpr int kKeys = 64;                // keys of a step
constexpr int kGroups = kTile / 16;      // scale groups of a key tile
constexpr int kStepGroups = kKeys / 16;
constexpr int kSoftmaxWarps = 4;         // per query tile
constexpr int kConvWarps = 4;
constexpr int kLoaderWarp = 2 * kSoftmaxWarps + kConvWarps;
constexpr int kIssueWarp = kLoaderWarp + 1;
constexpr int kThreads = 16 * 32;         // four warpgroups; the last two warps only keep theirs whole
// Registers per thread: the launch gives 128 to each; the softmax groups hold a step's scores and P.
constexpr int kSoftmaxRegs = 160, kOtherRegs = 96;
static_assert(2 * kSoftmaxRegs + 2 * kOtherRegs <= 4 * (65536 / kThreads), "what setmaxnreg hands out was launched");
constexpr int kInfo = 4;                 // key tiles whose scales are held
constexpr float kPScaleLog2 = 8.f;       // P = 2^8 of a row's largest: 11 bits down to 2^-22 of that
constexpr float kSlack = 5.f;            // maxima may be stale by 2^5: P < 2^14
// What a value scale counts as, and mw is above m at least: factors stay floats.
constexpr float kLeastLog2 = -120.f, kMostLog2 = 122.f;
constexpr int kSubTile = kTile * 128;    // 128 rows of 64 f16

struct TileInfo {
  float f[kGroups];     // key scale
  float w[kGroups];     // value scale
  float lw[kGroups];    // log2 of it, -infinity where it is 0 or no number
  float back[kGroups];  // its inverse (kRoundedSum)
  float least[2];       // per step: the smallest value scale, 0 if one is no number (kRoundedSum)
  uint32_t there;       // bit per group: the block exists and has keys that some row sees
  uint32_t pad;
};

template <int D>
struct Smem {
  static constexpr int kSub = D / 64;
  static constexpr int kOp = kSub * kSubTile;       // a [128 x D] f16 operand
  static constexpr int kRaw = kTile * D;            // a tile of levels
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kOp;           // two buffers
  static constexpr int kV = kK + 2 * kOp;           // two buffers
  static constexpr int kRawK = kV + 2 * kOp;
  static constexpr int kRawV = kRawK + kRaw;
  static constexpr int kInfoAt = kRawV + kRaw;
  static constexpr int kBars = kInfoAt + kInfo * static_cast<int>(sizeof(TileInfo));
  // q_full[2], raw_full[2], raw_free[2], op_full[2][2], op_free[2][2], s_full[2][2], p_full[2][2], pv_done[2][2],
  // info_full[4]
  static constexpr int kNumBars = 26 + kInfo;
  static constexpr int kMisc = kBars + kNumBars * 8;
  static constexpr int kTotal = kMisc + 16;
  static constexpr int kDynamic = kTotal + 1024;
};
static_assert(Smem<128>::kDynamic <= 227 * 1024, "shared memory of one SM");

__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// A from TMEM: lane = row, a 32-bit column holds two consecutive k.
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// D f32, A and B f16, B MN-major with bit 16; N >> 3 at [17, 23), M >> 4 at [24, 29).
__host__ __device__ constexpr uint32_t f16_idesc(int n, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? (1u << 16) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kTile >> 4) << 24);
}
// MN-major operand, 128-byte swizzle: rows are k indices of 64 n, groups of 8 rows 1024 bytes apart, the next 64 n
// one sub-tile further.
__device__ __forceinline__ uint64_t mn_major_desc(uint32_t addr) {
  uint64_t d = (addr & 0x3FFFF) >> 4;
  d |= static_cast<uint64_t>(kSubTile >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// The wait for loads in flight, tied to the registers of one of them: nothing that reads them moves before it.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
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
// Maxima that are NaN when one of their operands is.
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max16(const uint32_t* s) {
  auto f = [&](int i) { return __uint_as_float(s[i]); };
  const float a = max3(f(0), f(1), f(2)), b = max3(f(3), f(4), f(5)), c = max3(f(6), f(7), f(8));
  const float d = max3(f(9), f(10), f(11)), e = max3(f(12), f(13), f(14));
  return max2(max3(a, b, c), max3(d, e, f(15)));
}
// 2^x for a pair on the FMA pipe: x = n + f with |f| <= 1/2 by adding 1.5 2^23, a polynomial of degree 5 in f (the
// minimax one, relative error 2^-22.6, 2^-22.1 with the roundings), n into the exponent.  Below 2^-125 the result stays
// there, and for NaN it is there too: the kernel does not count on this to show one.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  x = pair(fmaxf(a, -125.f), fmaxf(b, -125.f));
  const uint64_t magic = pair(12582912.f, 12582912.f), minus = pair(-12582912.f, -12582912.f);
  const uint64_t r = add2(x, magic);
  const uint64_t f = fma2(add2(r, minus), pair(-1.f, -1.f), x);
  uint64_t y = pair(1.327647129073739e-3f, 1.327647129073739e-3f);
  y = fma2(y, f, pair(9.675540961325169e-3f, 9.675540961325169e-3f));
  y = fma2(y, f, pair(5.550713092088699e-2f, 5.550713092088699e-2f));
  y = fma2(y, f, pair(2.4022120237350464e-1f, 2.4022120237350464e-1f));
  y = fma2(y, f, pair(6.931469440460205e-1f, 6.931469440460205e-1f));
  y = fma2(y, f, pair(1.0000001192092896f, 1.0000001192092896f));
  float n0, n1;
  unpair(r, n0, n1);
  unpair(y, a, b);
  return pair(__uint_as_float(__float_as_uint(a) + (__float_as_uint(n0) << 23)),
              __uint_as_float(__float_as_uint(b) + (__float_as_uint(n1) << 23)));
}
// Scores of one row and step -> P in TMEM and the row's sum.  EDGE: some keys are hidden from some rows.
// `left` keys are visible from the step's first on; groups that are not `present` are not.
constexpr uint32_t kOnFma = 0x22;  // of the eight pairs of a group, those whose exp2 is a polynomial
// ROUNDED: the row's sum is that of P as f16 holds it (divided by its value scale again), so that the rounding of the
// largest ones cancels where the output is divided by it.  For f16 results only: their error falls from 0.00029 (up to
// 0.00032, 1.5 roundings, in batches with few prompts) to 0.00023 - 0.00025, for 10 % of the time (4 prompts 127 -> 140 us); with the
// sum corrected by what the rounding took, at edges too, 148 us.
template <bool EDGE, bool ROUNDED>
__device__ __forceinline__ void softmax_step(const uint32_t* s, const float* fs, const float* ws, const float* back,
                                             float rmul, float off, float unit, float per_unit, uint32_t t_p, int left,
                                             uint32_t present, uint64_t* sum) {
  const uint64_t off2 = pair(off, off);
#pragma unroll
  for (int cc = 0; cc < kKeys / 32; ++cc) {
    uint32_t w[16];
#pragma unroll
    for (int g = cc * 2; g < cc * 2 + 2; ++g) {
      const float f = fs[g] * rmul, vw = ws[g] * unit, vb = ROUNDED ? back[g] * per_unit : 0.f;
      const uint64_t f2 = pair(f, f), w2 = pair(vw, vw), back2 = pair(vb, vb);
      const int see = EDGE ? ((present >> g & 1) ? left - g * 16 : 0) : 16;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float a, b;
        const uint64_t x = fma2(pair(__uint_as_float(s[g * 16 + 2 * e]), __uint_as_float(s[g * 16 + 2 * e + 1])), f2, off2);
        if (!EDGE && (kOnFma >> e & 1)) {
          unpair(exp2_pair(x), a, b);
        } else {
          unpair(x, a, b);
          a = exp2_approx(a);
          b = exp2_approx(b);
        }
        if (EDGE) {
          if (2 * e >= see) a = 0.f;
          if (2 * e + 1 >= see) b = 0.f;
        }
        const uint64_t ab = pair(a, b);
        if constexpr (!ROUNDED) sum[e & 1] = add2(sum[e & 1], ab);
        unpair(mul2(ab, w2), a, b);
        if (EDGE) {  // 0 whatever the scale is
          if (2 * e >= see) a = 0.f;
          if (2 * e + 1 >= see) b = 0.f;
        }
        const uint32_t word = pack2(a, b, __half());
        if constexpr (ROUNDED) {
          float ra, rb;
          unpack2(word, ra, rb, __half());
          sum[e & 1] = fma2(pair(ra, rb), back2, sum[e & 1]);
        }
        w[(g & 1) * 8 + e] = word;
      }
    }
    tmem_st_x16(t_p + cc * 16, w);
  }
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ int rows_of(const Kv8AttentionParams& p, int q_len) {
  return min(max(q_len, 0), p.max_q) * (p.q_heads / p.cache.kv_heads);  // max_q * group fits
}
// Blocks of 256 rows that a request has here: none if its rows are few, none for rows behind the batch.
__device__ __forceinline__ int blocks_of(const Kv8AttentionParams& p, int q_len, int start, int min_rows) {
  if (rows_of(p, q_len) <= min_rows) return 0;
  const int64_t left = p.tokens - start;
  const int rows = rows_of(p, left < q_len ? static_cast<int>(max(left, static_cast<int64_t>(0))) : q_len);
  return (rows + 2 * kTile - 1) / (2 * kTile);
}

// Position of the n-th set bit (from 0), found by a converged warp.
__device__ __forceinline__ int nth_bit(uint32_t mask, int n, int lane) {
  const bool it = (mask >> lane & 1) && __popc(mask & ((1u << lane) - 1)) == n;
  return __ffs(__ballot_sync(~0u, it)) - 1;
}

// What CTA `index` works on: 256 query rows of a kv head of a request.
struct Item {
  int r, head, row0, rows;
  int keys;        // that its last row sees
  int64_t tok0;    // row of q of the request's first token
  int64_t behind;  // token i sees behind + i keys
};
// Heads vary fastest, then requests; of a request its last rows, with the most keys, come first: item by item through
// the list of (block from high to low, request that has it).  The host knows the rows of the batch only, which bound
// the list; a grid of requests x longest instead starts CTAs for nothing (64 single tokens and a prompt of 500 over
// 4 000 keys, 32 over 8 heads: 500 -> 180 us).  A converged warp; false: the list is shorter.
__device__ __forceinline__ bool item_of(const Kv8AttentionParams& p, uint32_t index, uint32_t blocks, int min_rows,
                                        int lane, Item& it) {
  const uint32_t KH = p.cache.kv_heads;
  int nth = static_cast<int>(index / KH);
  it.head = static_cast<int>(index % KH);
  // up to 32 requests: a lane per request has all that is needed of it, one load latency in all
  int my_len = 0, my_kv = 0, my_start = 0, my_blocks = 0;
  if (p.requests <= 32 && lane < p.requests) {
    my_len = p.q_lens[lane];
    my_kv = p.kv_lens[lane];
    my_start = p.q_start[lane];
    my_blocks = blocks_of(p, my_len, my_start, min_rows);
  }
  int block = -1, r = 0, q_asked, kv_have;
  if (p.requests <= 32) {
    // runs of blocks that the same requests have
    int b = static_cast<int>(__reduce_max_sync(~0u, static_cast<uint32_t>(my_blocks))) - 1;
    while (b >= 0) {
      const uint32_t m = __ballot_sync(~0u, my_blocks > b);
      const int low = static_cast<int>(__reduce_max_sync(~0u, my_blocks > b ? 0u : static_cast<uint32_t>(my_blocks)));
      const int c = __popc(m), n = (b - low + 1) * c;
      if (nth < n) {
        const int down = nth / c;
        block = b - down;
        r = nth_bit(m, nth - down * c, lane);
        break;
      }
      nth -= n;
      b = low - 1;
    }
    if (block < 0) return false;
    q_asked = __shfl_sync(~0u, my_len, r);
    kv_have = __shfl_sync(~0u, my_kv, r);
    it.tok0 = __shfl_sync(~0u, my_start, r);
  } else {
    auto blocks_at = [&](int i) {  // of request i + lane
      return i + lane < p.requests ? blocks_of(p, p.q_lens[i + lane], p.q_start[i + lane], min_rows) : 0;
    };
    // 32 blocks at a time, one per lane: how many requests have it
    for (int top = static_cast<int>(blocks) - 1; top >= 0 && block < 0; top -= 32) {
      const int levels = min(top, 31) + 1;
      int have = 0;
#pragma unroll 1
      for (int i = 0; i < p.requests; i += 32) {
        const int n = blocks_at(i);
        uint32_t m = __ballot_sync(~0u, n > top + 1 - levels);
        if (__popc(m) > levels) {
          for (int k = 0; k < levels; ++k) {
            const int c = __popc(__ballot_sync(~0u, n > top - k));
            if (lane == k) have += c;
          }
        } else {
          for (; m != 0; m &= m - 1) have += __shfl_sync(~0u, n, __ffs(m) - 1) > top - lane;
        }
      }
      if (lane >= levels) have = 0;
      int upto = have;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += u;
      }
      const uint32_t behind = __ballot_sync(~0u, upto > nth);
      const int at = behind != 0 ? __ffs(behind) - 1 : 31;
      if (behind != 0) block = top - at;
      nth -= __shfl_sync(~0u, behind != 0 ? upto - have : upto, at);
    }
    if (block < 0) return false;
#pragma unroll 1
    for (int i = 0; i < p.requests; i += 32) {
      const uint32_t m = __ballot_sync(~0u, blocks_at(i) > block);
      if (nth < __popc(m)) {
        r = i + nth_bit(m, nth, lane);
        break;
      }
      nth -= __popc(m);
    }
    q_asked = p.q_lens[r];
    kv_have = p.kv_lens[r];
    it.tok0 = p.q_start[r];
  }
  it.r = r;
  it.row0 = block * 2 * kTile;
  it.rows = min(2 * kTile, rows_of(p, q_asked) - it.row0);
  const int kv_len = min(max(kv_have, 0), p.table_width * p.cache.block_size);
  it.behind = static_cast<int64_t>(kv_len) - max(q_asked, 0) + 1;
  const int G = p.q_heads / p.cache.kv_heads;
  it.keys = static_cast<int>(max(static_cast<int64_t>(0), it.behind + (it.row0 + it.rows - 1) / G));
  return true;
}

// The items whose keys n CTAs share, and what a share leaves of their rows (256 of each item).
struct Shares {
  uint32_t from, to, n;
  int64_t rows;  // (to - from) * 256
  float* o;      // [n][rows][dim], of weights that add up to one: nothing overflows on the way to the join
  float2* ml;    // [n][rows] maximum and sum
};

// Which items' keys are shared; a way of writing a row that is not needed would cost registers (2 to 9 %).
enum class Cut { kNone, kAll, kSome };

template <typename T, int D, Cut CUT>
__global__ void __launch_bounds__(kThreads, 1)
prefill_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
               const __grid_constant__ Kv8AttentionParams p, int min_rows, uint32_t blocks, Shares sh, int box_rows) {
  using L = Smem<D>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t base = smem_u32(smem);
  const uint32_t bars = base + L::kBars;
  auto bar = [&](int i, int j) { return bars + 8u * (2 * i + j); };
  auto q_full = [&](int q) { return bar(0, q); };
  auto raw_full = [&](int v) { return bar(1, v); };
  auto raw_free = [&](int v) { return bar(2, v); };
  auto op_full = [&](int v, int b) { return bar(3 + v, b); };
  auto op_free = [&](int v, int b) { return bar(5 + v, b); };
  // of query tile q and step u (two buffers)
  auto s_full = [&](int q, int u) { return bar(7 + q, u & 1); };
  auto p_full = [&](int q, int u) { return bar(9 + q, u & 1); };
  auto pv_done = [&](int q, int u) { return bar(11 + q, u & 1); };
  auto info_full = [&](int i) { return bars + 8u * (26 + i); };
  TileInfo* info = reinterpret_cast<TileInfo*>(smem + L::kInfoAt);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  const int warp = __shfl_sync(~0u, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const Kv8Cache& c = p.cache;
  const int bs = c.block_size, G = p.q_heads / c.kv_heads;

  grid_dep_wait();
  grid_dep_launch();
  uint32_t index = blockIdx.x, share = 0, shares = 1;
  constexpr bool SHARES = CUT != Cut::kNone;
  constexpr bool kRoundedSum = std::is_same<T, __half>::value;
  if constexpr (CUT == Cut::kAll) {
    shares = sh.n;
    share = index % shares;
    index /= shares;
  } else if (SHARES && index >= sh.from) {
    index -= sh.from;
    const uint32_t span = (sh.to - sh.from) * sh.n;
    if (index < span) {
      shares = sh.n;
      share = index % shares;
      index = sh.from + index / shares;
    } else {
      index += sh.to - span;
    }
  }
  Item it;
  if (!item_of(p, index, blocks, min_rows, lane, it)) return;
  const int head = it.head, r = it.r, row0 = it.row0, rows = it.rows, keys = it.keys;
  const int64_t behind = it.behind, tok0 = it.tok0;
  // this CTA's share of the key tiles: nt tiles from key_first on, nu steps
  const int tiles_all = (keys + kTile - 1) / kTile;
  const int t_first = SHARES ? static_cast<int>(static_cast<int64_t>(tiles_all) * share / shares) : 0;
  const int nt = SHARES ? static_cast<int>(static_cast<int64_t>(tiles_all) * (share + 1) / shares) - t_first : tiles_all;
  const int key_first = t_first * kTile;
  const int nu = ((SHARES ? min(keys - key_first, nt * kTile) : keys) + kKeys - 1) / kKeys;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full(i), kSoftmaxWarps);
      mbar_init(raw_full(i), 1);
      mbar_init(raw_free(i), kConvWarps);
      for (int v = 0; v < 2; ++v) {
        mbar_init(s_full(v, i), 1);
        mbar_init(p_full(v, i), kSoftmaxWarps);
        mbar_init(pv_done(v, i), 1);
        mbar_init(op_full(v, i), kConvWarps);
        mbar_init(op_free(v, i), 2);
      }
    }
    for (int i = 0; i < kInfo; ++i) mbar_init(info_full(i), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kIssueWarp) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, *tmem_slot, 0);
  auto wait = [&](uint32_t b, uint32_t parity, int code) {
    return mbar_wait(b, parity, abort_flag, &g_kv8_prefill_status, code);
  };

  if (warp < 2 * kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------------------------ softmax: a thread per row
    const int q = warp / kSoftmaxWarps;
    const int row = (warp % kSoftmaxWarps) * 32 + lane;
    const int my_row = row0 + q * kTile + row;
    const bool valid = q * kTile + row < rows;
    const int i_tok = my_row / G, h = my_row % G;
    const int64_t at = tok0 + i_tok;
    const bool there = valid && at >= 0 && at < p.tokens;
    // a row that is not there computes along and is not stored
    const int lim = there ? static_cast<int>(max(static_cast<int64_t>(0), behind + i_tok)) : INT32_MAX;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp % kSoftmaxWarps) * 32) << 16);
    const uint32_t t_o = t_lane + 256 + q * D;
    const bool active = q * kTile < rows;
    // Rows of q come, and those of the output go, through the tile of q in shared memory: piece i of a warp's 32 rows
    // is kAtOnce rows, one 16-byte chunk per lane.
    constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;
    const int chunk = lane % kLanes;
    auto stage = [&](int r, int c) {
      return smem + L::kQ + q * L::kOp + (c / 8) * kSubTile + r * 128 + (((c % 8) ^ (r & 7)) << 4);
    };
    auto staged = [&](int i) { return stage((warp % kSoftmaxWarps) * 32 + i * kAtOnce + lane / kLanes, chunk); };
    float mul = 1.f;
    if (active && nt > 0) {
      // whole rows by neighbouring lanes, all loads before the first use
      const int64_t from = there ? at * p.ld_q + (head * G + h) * D : -1;
      uint4 w[kLanes];
#pragma unroll
      for (int i = 0; i < kLanes; ++i) {
        const int64_t f = __shfl_sync(~0u, from, i * kAtOnce + lane / kLanes);
        w[i] = f >= 0 ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + f + chunk * 8) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kLanes; ++i) {
        if constexpr (!std::is_same<T, __half>::value) {
          uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w}, top = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, max(x[e] & 0x7fffu, x[e] >> 16 & 0x7fffu));
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
          const float k = row_power(top << 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a, b;
            unpack2(x[e], a, b, T());
            x[e] = pack2(a * k, b * k, __half());
          }
          w[i] = make_uint4(x[0], x[1], x[2], x[3]);
          const float mine = __shfl_sync(~0u, k, lane % kAtOnce * kLanes);
          if (lane / kAtOnce == i) mul = mine;
        }
        *reinterpret_cast<uint4*>(staged(i)) = w[i];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full(q));
    }
    const float rmul = p.scale * 1.4426950408889634f / mul;
    // the first step in which some row of this warp does not see every key
    const int first_masked = (__reduce_min_sync(~0u, lim) - key_first) / kKeys;
    float m = -INFINITY;   // maximum of log2 p, and
    float mw = -INFINITY;  // of log2 p + log2 of its value scale: O is in units of 2^mw
    float unit = 0.f, per_unit = 0.f;  // 2^(m - mw) and its inverse
    uint64_t sum[2] = {0, 0};  // four partial sums
    bool ok = true;
    for (int u = 0; u < nu && active; ++u) {
      const int t = u >> 1, first_group = (u & 1) * kStepGroups;
      if ((u & 1) == 0) ok = wait(info_full(t % kInfo), (t / kInfo) & 1, 51);
      ok = ok && wait(s_full(q, u), (u >> 1) & 1, 52);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      tc_fence_after();
      const TileInfo& in = info[t % kInfo];
      const uint32_t t_s = t_lane + q * kTile + (u & 1) * kKeys;
      uint32_t s[kKeys];
#pragma unroll
      for (int cc = 0; cc < kKeys / 32; ++cc) tmem_ld_x32(t_s + cc * 32, s + cc * 32);
      float fs[kStepGroups], ws[kStepGroups], lw[kStepGroups];
#pragma unroll
      for (int g = 0; g < kStepGroups; ++g) {
        fs[g] = in.f[first_group + g];
        ws[g] = in.w[first_group + g];
        lw[g] = in.lw[first_group + g];
      }
      const uint32_t present = in.there >> first_group & ((1u << kStepGroups) - 1);
      const bool edge = u >= first_masked || present != (1u << kStepGroups) - 1;
      const int key0 = key_first + u * kKeys;
#pragma unroll
      for (int cc = 0; cc < kKeys / 32; ++cc) tmem_ld_wait32(s + cc * 32);
      float mx = -INFINITY, tx = -INFINITY;
      if (!edge) {
#pragma unroll
        for (int g = 0; g < kStepGroups; ++g) {
          const float top = max16(s + g * 16) * fs[g];
          mx = max2(mx, top);
          tx = fmaxf(tx, fmaf(top, rmul, lw[g]));
        }
      } else {
#pragma unroll
        for (int g = 0; g < kStepGroups; ++g) {
          const int see = (present >> g & 1) ? lim - key0 - g * 16 : 0;
          float top = -INFINITY;
#pragma unroll
          for (int e = 0; e < 16; ++e) top = e < see ? max2(top, __uint_as_float(s[g * 16 + e])) : top;
          mx = see > 0 ? max2(mx, top * fs[g]) : mx;
          tx = see > 0 ? fmaxf(tx, fmaf(top * fs[g], rmul, lw[g])) : tx;
        }
      }
      mx *= rmul;
      const float mn = fmaxf(m, mx);
      float wn = fmaxf(mw, tx);
      const bool up = mn > m + kSlack || wn > mw + kSlack;
      if (__any_sync(~0u, up)) {
        float a = 1.f;  // a row that stays keeps its maxima
        if (up) {
          const float k = exp2_approx(m - mn);
          sum[0] = mul2(sum[0], pair(k, k));
          sum[1] = mul2(sum[1], pair(k, k));
          if (wn > -INFINITY) {  // else its values so far are zeros
            wn = fmaxf(wn, mn + kLeastLog2);  // the largest p may belong to a block without values
            a = exp2_approx(mw - wn);
            unit = exp2f(mn - wn);
            per_unit = exp2f(wn - mn);
          }
          m = mn;
          mw = wn;
        }
        if (u > 0) {
          ok = wait(pv_done(q, u - 1), ((u - 1) >> 1) & 1, 65);  // nothing is being added to O
          ok = __all_sync(~0u, ok);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int cc = 0; cc < D / 16; ++cc) {
            uint32_t o[16];
            tmem_ld_x16(t_o + cc * 16, o);
            tmem_ld_wait_regs(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
            tmem_st_x16(t_o + cc * 16, o);
          }
        }
      }
      // A score that is NaN or +infinity makes all of the row's probabilities NaN, from here on: exp2_pair alone would
      // lose it where only its keys have one.
      if (!(mx < INFINITY)) m = __uint_as_float(0x7fc00000u);
      const float off = kPScaleLog2 - (m == -INFINITY ? 0.f : m);
      const float* back = in.back + first_group;
      // P stands for its part of the sum where what f16 cannot hold of it is nothing beside that
      const bool rounded = kRoundedSum && __all_sync(~0u, in.least[u & 1] * unit >= 0.0625f);
      if (edge) {
        softmax_step<true, false>(s, fs, ws, back, rmul, off, unit, per_unit, t_s, lim - key0, present, sum);
      } else if (kRoundedSum && rounded) {
        softmax_step<false, kRoundedSum>(s, fs, ws, back, rmul, off, unit, per_unit, t_s, 0, 0, sum);
      } else {
        softmax_step<false, false>(s, fs, ws, back, rmul, off, unit, per_unit, t_s, 0, 0, sum);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full(q, u));
    }
    // ---- epilogue
    if (active) {
      T* dst = static_cast<T*>(p.out) + (there ? at * p.ld_out + (head * G + h) * D : 0);
      const bool joined = CUT == Cut::kAll || (SHARES && shares > 1);
      const int64_t slot = SHARES ? share * sh.rows + (index - sh.from) * (2 * kTile) + q * kTile + row : 0;
      if (nt == 0) {
        if (there && joined) {
          sh.ml[slot] = make_float2(-INFINITY, 0.f);
        } else if (there) {
#pragma unroll
          for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
        }
      } else {
        if (ok) ok = wait(pv_done(q, nu - 1), ((nu - 1) >> 1) & 1, 53);
        ok = __all_sync(~0u, ok);
        if (ok) {
          tc_fence_after();
          float a, b;
          unpair(add2(sum[0], sum[1]), a, b);
          const float l = a + b;
          // 2^(mw - m) / l, over 2^16 at a time so that neither end passes the range of floats before the other
          const float k = l == 0.f || mw == -INFINITY ? 0.f : exp2f(mw - m - 16.f) / (l * 0x1p-16f);
          if (there && joined) sh.ml[slot] = make_float2(m, l);
          // the scores of all steps are done with q: its tile takes the output, f32 in two halves
          const int64_t to = !there ? -1 : joined ? slot * D : at * p.ld_out + (head * G + h) * D;
          auto emit = [&](auto f32) {
            constexpr bool F32 = decltype(f32)::value;
#pragma unroll
            for (int half = 0; half < (F32 ? 2 : 1); ++half) {
#pragma unroll
              for (int sub = 0; sub < D / 64; ++sub) {
#pragma unroll
                for (int e = 0; e < (F32 ? 1 : 2); ++e) {
                  const int cc = F32 ? half * (D / 64) + sub : sub * 2 + e;
                  uint32_t o[32];
                  tmem_ld_x32(t_o + cc * 32, o);
                  tmem_ld_wait32(o);
#pragma unroll
                  for (int j = 0; j < 32; ++j) o[j] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(o[j]) * k);
                  if constexpr (F32) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                      *reinterpret_cast<uint4*>(stage(row, sub * 8 + j / 4)) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                  } else {
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                      w[j] = pack2(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]), T());
#pragma unroll
                    for (int j = 0; j < 16; j += 4)
                      *reinterpret_cast<uint4*>(stage(row, cc * 4 + j / 4)) = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
                  }
                }
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < kLanes; ++i) {
                const int64_t f = __shfl_sync(~0u, to, i * kAtOnce + lane / kLanes);
                const uint4 x = *reinterpret_cast<const uint4*>(staged(i));
                if (f >= 0) {
                  if constexpr (F32) *reinterpret_cast<uint4*>(sh.o + f + half * (D / 2) + chunk * 4) = x;
                  else *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + f + chunk * 8) = x;
                }
              }
              __syncwarp();
            }
          };
          if constexpr (CUT != Cut::kSome) emit(std::bool_constant<SHARES>());
          else if (joined) emit(std::true_type());
          else emit(std::false_type());
        }
      }
    }
  } else {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp < kLoaderWarp) {
    // ------------------------------------------------------------------ converters: 32 keys of a tile per warp
    const int w = warp - 2 * kSoftmaxWarps;
    const int piece = lane & 3;
    bool ok = true;
    for (int t = 0; t < nt && ok; ++t) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int b = t & 1;
        ok = wait(raw_full(v), t & 1, 54);
        if (ok && t >= 2) ok = wait(op_free(v, b), ((t >> 1) - 1) & 1, 55);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        const uint8_t* src = smem + (v ? L::kRawV : L::kRawK);
        uint8_t* dst = smem + (v ? L::kV : L::kK) + b * L::kOp;
        // a quarter warp reads four 16-byte pieces of two keys and writes them as 32 bytes each; which half of a
        // 128-value row it takes alternates with the key, so that neither side meets in a bank
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = D == 128 ? w * 32 + j * 8 + (lane >> 3) * 2 + ((lane >> 2) & 1) : w * 32 + j * 8 + (lane >> 2);
#pragma unroll
          for (int i = 0; i < L::kSub; ++i) {
            const int sub = D == 128 ? i ^ (key & 1) : 0;
            const uint4 x = *reinterpret_cast<const uint4*>(
                D == 128 ? src + key * 128 + (((sub * 4 + piece) ^ (key & 7)) << 4)
                         : src + key * 64 + ((piece ^ ((key >> 1) & 3)) << 4));
            uint32_t y[8];
            const uint32_t in4[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[2 * e] = bytes_to_f16(in4[e], 0x4140);
              y[2 * e + 1] = bytes_to_f16(in4[e], 0x4342);
            }
            uint8_t* o = dst + sub * kSubTile + key * 128;
            *reinterpret_cast<uint4*>(o + (((2 * piece) ^ (key & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<uint4*>(o + (((2 * piece + 1) ^ (key & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(op_full(v, b));
          mbar_arrive(raw_free(v));
        }
      }
    }
  } else if (warp == kLoaderWarp) {
    // ------------------------------------------------------------------ loader: lane g < 8 knows group g of the tile
    bool ok = true;
    auto block_of = [&](int t) {  // -1: no such block, or no key of the group is seen
      const int key = key_first + t * kTile + lane * 16;
      int id = -1;
      if (t < nt && lane < kGroups && key < keys) {
        const int b = p.table[static_cast<int64_t>(r) * p.table_width + key / bs];
        if (b >= 0 && b < c.num_blocks) id = b;
      }
      return id;
    };
    const int boxes = kTile / box_rows, per_box = box_rows / 16;
    int id = block_of(0);
    for (int t = 0; t < nt; ++t) {
      const int box_id = __shfl_sync(~0u, id, (lane * per_box) & 31);
      const bool mine = lane < boxes && box_id >= 0;
      const uint32_t bytes = __popc(__ballot_sync(~0u, mine)) * box_rows * D;
      const int off = (t * kTile + lane * box_rows) & (bs - 1);
      if (t > 0) ok = wait(raw_free(0), (t - 1) & 1, 56);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(raw_full(0), bytes);
      __syncwarp();
      if (mine) tma_load_3d(base + L::kRawK + lane * box_rows * D, &tk, raw_full(0), 0, off, box_id * c.kv_heads + head);
      // while the keys are on their way: the scales, and the blocks of the next tile
      float ks = 0.f, vs = 0.f;
      if (id >= 0) {
        ks = c.k_scale[static_cast<int64_t>(id) * c.kv_heads + head];
        vs = c.v_scale[static_cast<int64_t>(id) * c.kv_heads + head];
      }
      const int id_next = block_of(t + 1);
      if (t > 0) ok = wait(raw_free(1), (t - 1) & 1, 57);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(raw_full(1), bytes);
      __syncwarp();
      if (mine) tma_load_3d(base + L::kRawV + lane * box_rows * D, &tv, raw_full(1), 0, off, box_id * c.kv_heads + head);
      // Tile t - 4, whose entry this overwrites, is done with: the keys of tile t - 1 are converted, into the buffer
      // of tile t - 3, so the scores of its second step were complete, and they were begun when P V of the second
      // step of tile t - 4 was, for which its entry was read.
      const uint32_t there = __ballot_sync(~0u, id >= 0);
      TileInfo& in = info[t % kInfo];
      if (lane < kGroups) {
        in.f[lane] = ks;
        in.w[lane] = vs;
        in.lw[lane] = vs > 0.f && vs < INFINITY ? fminf(fmaxf(__log2f(vs), kLeastLog2), kMostLog2) : -INFINITY;
      }
      if (kRoundedSum) {
        float least = vs >= 0.f && vs < INFINITY ? vs : 0.f;
        least = fminf(least, __shfl_xor_sync(~0u, least, 1));
        least = fminf(least, __shfl_xor_sync(~0u, least, 2));
        if (lane < kGroups) {
          in.back[lane] = 1.f / vs;
          if (lane % kStepGroups == 0) in.least[lane / kStepGroups] = least;
        }
      }
      if (lane == 0) in.there = there;
      __syncwarp();
      if (lane == 0) mbar_arrive(info_full(t % kInfo));
      id = id_next;
    }
  } else if (warp < kIssueWarp + 2) {
    // ------------------------------------------------------------------ issuers: one warp per query tile
    const int q = warp - kIssueWarp;
    const bool active = q * kTile < rows;
    constexpr uint32_t idesc_s = f16_idesc(kKeys, false);
    constexpr uint32_t idesc_o = f16_idesc(D, true);
    bool ok = true;
    auto await = [&](uint32_t b, uint32_t parity, int code) { ok = __all_sync(~0u, ok && wait(b, parity, code)); };
    // S of step u, into the buffer that P of step u - 2 was in
    auto scores = [&](int u) {
      const int b = (u >> 1) & 1;
      if ((u & 1) == 0) await(op_full(0, b), (u >> 2) & 1, 59);
      if (active && u >= 2) await(pv_done(q, u), ((u >> 1) - 1) & 1, 61);
      if (!ok) return;
      tc_fence_after();
      const uint32_t q_at = base + L::kQ + q * L::kOp, k_at = base + L::kK + b * L::kOp + (u & 1) * kKeys * 128;
      if (elect_one()) {
        if (active) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t step = (kk >> 2) * kSubTile;
            umma_f16_ss(tmem + q * kTile + (u & 1) * kKeys, make_kmajor_sw128_desc(q_at + step) + 2 * (kk & 3),
                        make_kmajor_sw128_desc(k_at + step) + 2 * (kk & 3), idesc_s, kk != 0 ? 1u : 0u);
          }
          umma_commit(s_full(q, u));
          if ((u & 1) == 1) umma_commit(op_free(0, b));
        } else if ((u & 1) == 1) {  // the other tile alone decides when the operands are free
          mbar_arrive(op_free(0, b));
        }
      }
      __syncwarp();
    };
    auto products = [&](int u) {
      const int b = (u >> 1) & 1;
      if ((u & 1) == 0) await(op_full(1, b), (u >> 2) & 1, 62);
      if (active) await(p_full(q, u), (u >> 1) & 1, 63);
      if (!ok) return;
      tc_fence_after();
      const uint32_t v_at = base + L::kV + b * L::kOp + (u & 1) * kKeys * 128;
      const uint32_t t_p = tmem + q * kTile + (u & 1) * kKeys, t_o = tmem + 256 + q * D;
      if (elect_one()) {
        if (active) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            umma_f16_ts(t_o, t_p + kk * 8, mn_major_desc(v_at + kk * 16 * 128), idesc_o, (u | kk) != 0 ? 1u : 0u);
          umma_commit(pv_done(q, u));
          if ((u & 1) == 1) umma_commit(op_free(1, b));
        } else if ((u & 1) == 1) {
          mbar_arrive(op_free(1, b));
        }
      }
      __syncwarp();
    };
    if (active && nu > 0) await(q_full(q), 0, 58);
    for (int u = 0; u < 2 && u < nu && ok; ++u) scores(u);
    for (int u = 0; u < nu && ok; ++u) {
      products(u);
      if (ok && u + 2 < nu) scores(u + 2);
    }
  }
  }

  __syncwarp();
  if (*abort_flag) {  // let copies and products in flight end before shared memory and TMEM are given back
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the shares of the rows of the blockIdx.x-th item that has them: a warp per row, a lane per share for the weights.
constexpr int kJoinThreads = 256, kMostShares = 32, kMostPieces = 512;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
prefill_join_kernel(const __grid_constant__ Kv8AttentionParams p, int min_rows, uint32_t blocks, Shares sh) {
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, G = p.q_heads / p.cache.kv_heads, shares = static_cast<int>(sh.n);
  Item it;
  if (!item_of(p, sh.from + blockIdx.x, blocks, min_rows, lane, it)) return;
  for (int i = (blockIdx.y * kJoinThreads + threadIdx.x) / 32; i < it.rows; i += gridDim.y * (kJoinThreads / 32)) {
    const int64_t at = it.tok0 + (it.row0 + i) / G;
    if (at < 0 || at >= p.tokens) continue;
    const int col = it.head * G + (it.row0 + i) % G;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (2 * kTile) + i;
    const float2 ml = lane < shares ? sh.ml[lane * sh.rows + row] : make_float2(-INFINITY, 0.f);
    float top = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    // a share that saw no key has a sum of 0, and its output may not even be written
    float w = ml.y == 0.f ? 0.f : ml.y * exp2_approx(ml.x - top), sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    w = sum == 0.f ? 0.f : w / sum;
    constexpr int E = D / 32;
    float acc[E] = {};
#pragma unroll 8
    for (int k = 0; k < shares; ++k) {
      const float wk = __shfl_sync(~0u, w, k);
      const float* v = sh.o + (k * sh.rows + row) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 x = wk != 0.f ? *reinterpret_cast<const float2*>(v + e) : make_float2(0.f, 0.f);
        acc[e] += x.x * wk;
        acc[e + 1] += x.y * wk;
      }
    }
    uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + at * p.ld_out + col * D + lane * E);
#pragma unroll
    for (int e = 0; e < E; e += 2) out[e / 2] = pack2(acc[e], acc[e + 1], T());
  }
}

struct Launch {
  int64_t rows, blocks, items;
  Shares sh;
};
// The grid, and which items' keys are cut into shares: all of them, so that few rows over long caches fill the GPU, or
// those that would not fill the last round of CTAs.  As many shares as make one to three full rounds, where the rounds
// (2.1 us per key tile and 8 per CTA) and the join (5 us, and its bytes at 6 TB/s) come to 6 % less than they do without
// shares.  A round of 148 equal CTAs takes 2.6 us per key tile in f16 and 2.3 in bf16 at heads of 128, 2.3 and 2.0 at heads
// of 64: one pair of figures serves both.  The host has bounds only: the rows of the batch, and the longest cache.
// One request, 8 kv heads with 4 query heads each, us without shares -> as chosen:
//                       128, f16        128, bf16       64, f16         64, bf16
//   64 over  8 000     162 ->   36     143 ->   35     155 ->   30     129 ->   26
//  100 over 30 000     579 ->   92     490 ->   83     559 ->   84     466 ->   68
//  200 over  3 000      70 ->   36      66 ->   37      62 ->   31      54 ->   29
//  512 over  8 192     167 ->  106     145 ->   95     156 ->   99     133 ->   85
//  700 over  2 500      61 ->   61      56 ->   61      54 ->   54      48 ->   48
// 1500 over 12 000     441 ->  365     377 ->  298     409 ->  324     350 ->  263
// 2048 over 30 000    1127 -> 1174     990 ->  995    1058 -> 1010     902 ->  826
Launch launch_of(const Kv8AttentionParams& p, void* workspace) {
  Launch l = {};
  const int64_t G = p.q_heads / p.cache.kv_heads, KH = p.cache.kv_heads, sms = device_sm_count();
  l.rows = p.max_q * G;
  l.blocks = (l.rows + 2 * kTile - 1) / (2 * kTile);
  // no more blocks than the rows of the batch make, and one more for the rest of each request
  l.items = std::min(l.blocks * p.requests, p.tokens * G / (2 * kTile) + std::min<int64_t>(p.requests, p.tokens)) * KH;
  const int64_t likely = std::min(l.items, (p.tokens * G + 2 * kTile - 1) / (2 * kTile) * KH);
  const double tiles = static_cast<double>((p.max_kv + kTile - 1) / kTile);
  auto rounds = [&](int64_t ctas, int64_t n) { return static_cast<double>((ctas + sms - 1) / sms) * (tiles / n * 2.1 + 8); };
  double best = 0.94 * rounds(likely, 1);
  l.sh.n = 1;
  for (const int64_t from : {int64_t{0}, likely / sms * sms}) {
    const int64_t cut = likely - from;
    for (int64_t round = 1; round <= 3 && cut > 0; ++round) {
      const int64_t n = std::min({round * sms / cut, int64_t{kMostShares}, static_cast<int64_t>(tiles) / 4});
      if (n < 2) continue;
      const double t = rounds(from, 1) + rounds(cut * n, n) + 5 + static_cast<double>(cut * n) * (2 * kTile) * p.cache.dim * 8 / 6e6;
      if (t < best) {
        best = t;
        l.sh.n = static_cast<uint32_t>(n);
        l.sh.from = static_cast<uint32_t>(from);
      }
    }
  }
  if (l.sh.n > 1) {
    l.sh.to = static_cast<uint32_t>(std::min<int64_t>(l.items, l.sh.from + kMostPieces / l.sh.n));
    l.sh.rows = static_cast<int64_t>(l.sh.to - l.sh.from) * (2 * kTile);
    l.sh.o = static_cast<float*>(workspace);
    if (workspace) l.sh.ml = reinterpret_cast<float2*>(l.sh.o + l.sh.n * l.sh.rows * p.cache.dim);
  }
  return l;
}

template <typename T, int D>
cudaError_t launch_t(const Kv8AttentionParams& p, int min_rows, const Launch& l, cudaStream_t stream, const char** err) {
  if (l.rows > INT32_MAX - 2 * kTile || l.items > INT32_MAX / 2) {
    *err = "too many query rows";
    return cudaErrorInvalidValue;
  }
  CUtensorMap tk, tv;
  const int box = p.cache.block_size < kTile ? p.cache.block_size : kTile;
  if (!make_map(&tk, p.cache.k, p.cache, box) || !make_map(&tv, p.cache.v, p.cache, box)) {
    *err = "cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  const Cut cut = l.sh.n == 1 ? Cut::kNone : l.sh.from == 0 && l.sh.to == l.items ? Cut::kAll : Cut::kSome;
  auto kern = cut == Cut::kNone  ? prefill_kernel<T, D, Cut::kNone>
              : cut == Cut::kAll ? prefill_kernel<T, D, Cut::kAll>
                                 : prefill_kernel<T, D, Cut::kSome>;
  constexpr int smem = Smem<D>::kDynamic;
  static std::atomic<uint64_t> ready[3] = {{0}, {0}, {0}};
  const cudaError_t st = allow_smem(kern, smem, ready[static_cast<int>(cut)]);
  if (st != cudaSuccess) return st;
  const int64_t ctas = l.items + static_cast<int64_t>(l.sh.to - l.sh.from) * (l.sh.n - 1);
  return launch_dependent(kern, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), smem, stream, tk, tv, p, min_rows,
                          static_cast<uint32_t>(l.blocks), l.sh, box);
}

template <typename T, int D>
cudaError_t join_t(const Kv8AttentionParams& p, int min_rows, const Launch& l, cudaStream_t stream) {
  const int64_t items = l.sh.to - l.sh.from;  // two rounds of CTAs, a row per warp at least
  const int slices = static_cast<int>(std::clamp<int64_t>(16 * device_sm_count() / items, 1, 2 * kTile * 32 / kJoinThreads));
  return launch_dependent(prefill_join_kernel<T, D>, dim3(static_cast<unsigned>(items), slices), dim3(kJoinThreads), 0,
                          stream, p, min_rows, static_cast<uint32_t>(l.blocks), l.sh);
}

}  // namespace

int64_t kv8_prefill_workspace_bytes(const Kv8AttentionParams& p) {
  const Launch l = launch_of(p, nullptr);
  return l.sh.n > 1 ? l.sh.n * l.sh.rows * (static_cast<int64_t>(p.cache.dim) * 4 + 8) : 0;
}

cudaError_t kv8_prefill_launch(const Kv8AttentionParams& p, int min_rows, void* workspace, cudaStream_t stream,
                               const char** err) {
  const Launch l = launch_of(p, workspace);
  if (p.cache.dim == 128)
    return p.type == kKvF16 ? launch_t<__half, 128>(p, min_rows, l, stream, err)
                            : launch_t<__nv_bfloat16, 128>(p, min_rows, l, stream, err);
  return p.type == kKvF16 ? launch_t<__half, 64>(p, min_rows, l, stream, err)
                          : launch_t<__nv_bfloat16, 64>(p, min_rows, l, stream, err);
}

cudaError_t kv8_prefill_join_launch(const Kv8AttentionParams& p, int min_rows, void* workspace, cudaStream_t stream) {
  const Launch l = launch_of(p, workspace);
  if (l.sh.n == 1) return cudaSuccess;
  if (p.cache.dim == 128)
    return p.type == kKvF16 ? join_t<__half, 128>(p, min_rows, l, stream)
                            : join_t<__nv_bfloat16, 128>(p, min_rows, l, stream);
  return p.type == kKvF16 ? join_t<__half, 64>(p, min_rows, l, stream)
                          : join_t<__nv_bfloat16, 64>(p, min_rows, l, stream);
}

int kv8_status_fetch_and_clear() {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, g_kv8_prefill_status, sizeof(int)) != cudaSuccess) return -1;
  if (h != 0) {
    int z = 0;
    cudaMemcpyToSymbol(g_kv8_prefill_status, &z, sizeof(int));
  }
  return h;
}

}  // namespace disc_b200
