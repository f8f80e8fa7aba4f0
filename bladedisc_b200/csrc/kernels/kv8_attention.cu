// Attention over the 8-bit paged cache:
//   s_ij = scale * k_scale[block(j)] * (q_i . k_j),   j <= kv_len - q_len + i
//   o_i  = sum_j softmax(s_i)_j * v_scale[block(j)] * v_j,   0 where row i sees no key.
#include "kv8.h"

#include <algorithm>
#include <type_traits>

#include "device_info.h"
#include "kv8_attention.cuh"

namespace disc_b200 {

namespace {

// ------------------------------------------------------------------------------------------------ few rows
// Up to a few dozen query rows per request and kv head: the cache is read once and its bytes are what bounds the
// kernel, closely followed by the instructions that turn levels into f16.
//
// An item is a request, a kv head and 8 or 16 query rows (query heads of that kv head, tokens of that request); its work
// is steps of 32 keys.  All steps of all items are laid end to end and cut into equal shares, one per CTA, three CTAs
// per SM: ragged lengths balance to one step.  A share that ends inside an item leaves its partial maximum, sum and
// output in the workspace, and a second small kernel joins them.  Short caches (max_kv <= kKv8DirectKeys) take one CTA
// per item and need neither, and so do those up to kDirectMost keys when there are items for two rounds of CTAs: 32
// requests of up to 2048 tokens and 32 heads took 61 us that way and 73 in shares (before the second product below); 8
// requests of up to 32700 tokens and 8 kv heads 252 us that way and 61 in shares.
//
// Inside a CTA a warp runs by itself: it fetches its steps with 16-byte asynchronous copies into its own ring (TMA
// boxes of 2 to 4 KB cost the warp 170 cycles each, a quarter of a step), multiplies with mma.sync m16n8k16, keeps
// running maximum, sum and output in registers and meets the others at the end of the item.
//
//   S' = K Q'    keys are the wide operand, so that eight query rows fill the instruction (a decode step has one to
//                eight); the head dimension is permuted alike in K and Q so that a lane's fragments are the bytes of
//                16-byte loads; levels become f16 exactly (byte b as 0x6400 | b + 128 is 1152 + b, one subtraction).
//   O' += V' P'  a lane's fragments pair bytes of two keys: two byte permutes, again exact in f16; P changes its
//                fragment layout with one 8 x 8 transpose.
// Query rows in bf16 are scaled by a power of two per row to f16 (exact but for values 2^-24 of the row's largest).
// P, a probability times its value scale, goes to f16 as 2^11 for a row's largest, so that it keeps its 11 bits down to
// 2^-25 of that; a row of O is in units of the largest so far.  With f16 results what the
// rounding of P leaves out is multiplied too: over values of either sign it weighs as much as the rounding of the result
// (error 0.00021, that of one rounding, instead of 0.00025 to 0.00031; 61 -> 65 us for the 32 requests).  In bf16 results
// (0.0017) it does not show.
// Rows in the ring are swizzled (16-byte chunk c of row r at c ^ (r & 7), for dim 64 c ^ (r / 2 & 3)); that and the key
// order perm(n) = n ^ ((n & 1) << 2) make the 16-byte shared-memory reads free of bank conflicts.
//
// What bounds it: the cache's bytes.  On the GPU the 32 requests, 330 MB, take 65 us (5.1 TB/s, 0.77 of the measured copy
// rate); long contexts of 270 MB, 8 requests of up to 32700 tokens or one of 131072, 8 kv heads, 59 and 63 us (4.6 and
// 4.3 TB/s).  Without any arithmetic the copies of those took 54 and 57, of which 10 are the start of a share (sums, table,
// scales, first copy one after the other) and the join.  Measured for the 32 requests, then at 61 us, and not kept: four
// CTAs per SM with a ring of three tiles (65 us), levels as f16 subnormals in the first product (64).
constexpr int kStep = 32;         // keys per step of a warp
constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = kSplitWarps * 32;
constexpr int kSplitRows = 64;    // query rows per request and kv head up to which this kernel is the faster one
constexpr int kDirectMost = 4096;  // longest cache that is not cut when there are items for two rounds of CTAs
// The same with prompts in the batch: one tile of eight rows.  Requests of 9 to 64 rows go to the prompts' CTAs, one for
// all their keys.  Beside 3 prompts of 511 over 2 000 keys, 32 over 8 heads, that is right for 20 requests of 16 tokens
// (136 us; here 223) and even for 20 of 4 (156; 151), but not over long caches: one request of 4 tokens over 32 000 keys
// beside a prompt of 500 takes 263 us (here 93), a single token with 16 query heads per kv head 448 (78).
constexpr int kSplitRowsMixed = 8;
constexpr float kPScaleLog2 = 11.f;
constexpr float kMaxSlack = 2.f;  // maxima may be stale by this much (in log2) before O is rescaled: P < 2^14
constexpr float kNone = -3.4028235e38f;  // maximum of a row that has seen no key: below it, -infinity alone
// What a value scale counts as, and mw is above m at least: factors stay floats.
constexpr float kLeastLog2 = -120.f, kMostLog2 = 122.f;

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t w) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
  return r;
}

// Sixteen consecutive 16-bit values of a query row as f16 words; returns nothing for a row that is not there.
__device__ __forceinline__ void load_q16(const __half* p, bool there, float, uint32_t* w) {
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (there) {
    a = *reinterpret_cast<const uint4*>(p);
    b = *reinterpret_cast<const uint4*>(p + 8);
  }
  w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
}
__device__ __forceinline__ void load_q16(const __nv_bfloat16* p, bool there, float mul, uint32_t* w) {
  float f[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = 0.f;
  if (there) {
    load8(p, f);
    load8(p + 8, f + 8);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack2(f[2 * i] * mul, f[2 * i + 1] * mul, __half());
}
constexpr int kMaxRows = 16;  // of an item

// What is left of a share that ends inside an item: a maximum, a sum and an output per row.
struct SplitWs {
  float* o;      // [2 * ctas][rows][dim]: slot 2 c for a piece that does not start its item, 2 c + 1 for one that does
  float2* ml;    // [2 * ctas][rows]
  int4* desc;    // [ctas] {request, kv head, row tile, pieces} of the item that CTA c starts and does not finish
};

struct SplitShape {
  int stream;       // 1: equal shares of all steps; 0: one CTA per item
  int row_tiles;    // per kv head, from max_q (stream = 0)
  int max_rows;     // requests with more query rows per kv head than this are left to the other kernel
};

template <int D>
struct SplitSmem {
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kHalf = kStep * D;  // bytes of the keys (or values) of one step
  static constexpr int kRing = kSplitWarps * kStages * 2 * kHalf;
  static constexpr int kParts = kSplitWarps * kMaxRows * D * 4;  // O of every warp, in the place of the rings
  static constexpr int kDynamic = kRing > kParts ? kRing : kParts;
};

// Query rows (tokens x heads of a group) and steps of one request; no rows if the request is not for this kernel.
struct Request {
  int q_asked, q_len, kv_len, tiles, steps;
};
__device__ __forceinline__ Request request_of(const Kv8AttentionParams& p, int r, int max_rows, int tile_rows) {
  Request q;
  const int G = p.q_heads / p.cache.kv_heads;
  q.q_asked = max(p.q_lens[r], 0);
  q.q_len = min(q.q_asked, p.max_q);
  q.kv_len = min(max(p.kv_lens[r], 0), p.table_width * p.cache.block_size);
  const int rows = q.q_len * G <= max_rows ? q.q_len * G : 0;  // q_len <= max_q: fits
  q.tiles = static_cast<int>(static_cast<uint32_t>(rows + tile_rows - 1) / static_cast<uint32_t>(tile_rows));
  q.steps = max(1, (q.kv_len + kStep - 1) / kStep);
  return q;
}

template <typename T, int D, int NQ>
__device__ __forceinline__ void split_body(const Kv8AttentionParams& p, const SplitShape& shape, const SplitWs& ws) {
  using L = SplitSmem<D>;
  constexpr int W = kSplitWarps, S = L::kStages;
  constexpr int KQ = D / 16;  // k steps of the first product
  constexpr int NV = D / 16;  // m tiles of the second
  constexpr int ROWS = 8 * NQ;
  constexpr bool kRest = std::is_same<T, __half>::value;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float part_m[W][ROWS], part_l[W][ROWS];
  __shared__ long long sums[W];
  __shared__ int found[2];
  __shared__ long long found_at;

  const Kv8Cache& c = p.cache;
  const int bs = c.block_size, G = p.q_heads / c.kv_heads, KH = c.kv_heads;
  const int warp = __shfl_sync(~0u, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  // ---- which steps are this CTA's: `left` steps from step `s0` of item `item` of request r on
  int r, item, s0;
  int64_t left, total = 0;
  if (!shape.stream) {
    r = blockIdx.y;
    const Request q = request_of(p, r, shape.max_rows, ROWS);
    const int tile = blockIdx.x % shape.row_tiles;
    if (tile >= q.tiles) return;
    item = static_cast<int>(blockIdx.x / shape.row_tiles) * q.tiles + tile;
    s0 = 0;
    left = q.steps;
  } else {
    const int per = (p.requests + kSplitThreads - 1) / kSplitThreads;
    const int r0 = min(p.requests, static_cast<int>(threadIdx.x) * per), r1 = min(p.requests, r0 + per);
    int64_t mine = 0;
    for (int i = r0; i < r1; ++i) {
      const Request q = request_of(p, i, shape.max_rows, ROWS);
      mine += static_cast<int64_t>(q.tiles) * KH * q.steps;
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    for (int w = 0; w < W; ++w) {
      if (w < warp) incl += sums[w];
      total += sums[w];
    }
    const int64_t begin = total * blockIdx.x / gridDim.x, end = total * (blockIdx.x + 1) / gridDim.x;
    left = end - begin;
    if (left > 0 && begin >= incl - mine && begin < incl) {  // one thread's requests hold the first step
      int64_t at = incl - mine;
      for (int i = r0; i < r1; ++i) {
        const Request q = request_of(p, i, shape.max_rows, ROWS);
        const int64_t work = static_cast<int64_t>(q.tiles) * KH * q.steps;
        if (begin < at + work) {
          found[0] = i;
          found_at = begin - at;
          break;
        }
        at += work;
      }
    }
    if (threadIdx.x == 0) ws.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    __syncthreads();
    if (left <= 0) {  // nothing of an item that may go on around this CTA
      if (threadIdx.x < ROWS) ws.ml[2 * static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x] = make_float2(-INFINITY, 0.f);
      return;
    }
    r = found[0];
    const Request q = request_of(p, r, shape.max_rows, ROWS);
    item = static_cast<int>(found_at / q.steps);
    s0 = static_cast<int>(found_at % q.steps);
  }
  Request rq = request_of(p, r, shape.max_rows, ROWS);

  const uint8_t* ring_ptr = smem + warp * (S * 2 * L::kHalf);
  // where this lane's 16 bytes of every 512 go (dim 128: copies of even and odd index differ in the swizzle)
  const uint32_t ring = smem_u32(ring_ptr);
  const uint32_t put_even = D == 128 ? (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4)
                                     : (lane >> 2) * 64 + (((lane & 3) ^ (lane >> 3 & 3)) << 4);
  const uint32_t put_odd = D == 128 ? put_even ^ 64 : put_even;
  const int prow = g ^ ((g & 1) << 2);         // key of n = g in a group of eight
  const int v0 = 2 * t, v1 = (2 * t + 1) ^ 4;  // keys of this lane's columns

  while (left > 0) {
    while (item >= rq.tiles * KH) {  // on to the next request with rows
      if (++r >= p.requests) return;  // not with lengths that stay as they are during the call
      item = 0;
      rq = request_of(p, r, shape.max_rows, ROWS);
    }
    const int head = item / rq.tiles, tile = item % rq.tiles;
    const int s1 = static_cast<int>(min(static_cast<int64_t>(rq.steps), s0 + left));
    const int row0 = tile * ROWS;
    const int rows = min(ROWS, rq.q_len * G - row0);
    const int64_t tok0 = p.q_start[r];
    const int64_t behind = static_cast<int64_t>(rq.kv_len) - rq.q_asked + 1;
    // keys that the first row of the tile sees, and the last one
    const int lim_first = static_cast<int>(max(static_cast<int64_t>(0), behind + row0 / G));
    const int keys = static_cast<int>(max(static_cast<int64_t>(0), behind + (row0 + rows - 1) / G));

    // this warp's steps: first, first + W, ...
    const int first = static_cast<int>(s0) + warp;
    const int last = min(s1, (keys + kStep - 1) / kStep);
    const int mine = last > first ? (last - first + W - 1) / W : 0;

    // what a lane knows of half a step, 16 keys: half lane & 1 of step 16 * group + (lane >> 1)
    struct Info { int id; float ks, vs; } cur, next;
    auto lookup = [&](int base) {
      Info f;
      f.id = -1;
      f.ks = f.vs = 0.f;
      const int n = base + (lane >> 1);
      const int key = (first + n * W) * kStep + (lane & 1) * 16;
      if (n < mine && key < keys) {
        const int id = p.table[static_cast<int64_t>(r) * p.table_width + key / bs];
        if (id >= 0 && id < c.num_blocks) {
          f.id = id;
          f.ks = c.k_scale[static_cast<int64_t>(id) * KH + head];
          f.vs = c.v_scale[static_cast<int64_t>(id) * KH + head];
        }
      }
      return f;
    };
    // the whole warp copies step n into its stage: 32 keys and 32 values, 512 bytes per instruction
    auto issue = [&](int n, int id0, int id1) {
      const uint32_t kt = ring + (n % S) * (2 * L::kHalf);
      const int off = ((first + n * W) * kStep) & (bs - 1);  // 0 for blocks of 16, whose halves have a block each
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int id = h == 0 ? id0 : id1;
        if (id < 0) continue;
        const int64_t at = ((static_cast<int64_t>(id) * KH + head) * bs + (bs >= kStep ? off + h * 16 : 0)) * D + lane * 16;
        const int8_t* ks = c.k + at;
        const int8_t* vs = c.v + at;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint32_t to = kt + h * (L::kHalf / 2) + i * 512 + ((i & 1) ? put_odd : put_even);
          cp_async16(to, ks + i * 512);
          cp_async16(to + L::kHalf, vs + i * 512);
        }
      }
      cp_async_commit();
    };

    cur = lookup(0);
#pragma unroll
    for (int n = 0; n < S; ++n) {
      const int id0 = __shfl_sync(~0u, cur.id, 2 * n), id1 = __shfl_sync(~0u, cur.id, 2 * n + 1);
      issue(n, n < mine ? id0 : -1, n < mine ? id1 : -1);
    }
    next = lookup(16);

    // Q fragments, while the first keys are on their way: this lane loads row 8 j + g; its scores belong to the rows 8 j + 2 t + e
    uint32_t qb[NQ][KQ][2];
    // maximum of log2 p, sum of p, maximum of log2 p + log2 of its value scale (O is in units of 2^mw), 2^(m - mw)
    float qmul[NQ][2], m[NQ][2], l[NQ][2], mw[NQ][2], unit[NQ][2];
    int lim[NQ][2];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      const int row = j * 8 + g;
      const int i = (row0 + row) / G, h = (row0 + row) % G;
      const int64_t at = tok0 + i;
      const bool there = row < rows && at >= 0 && at < p.tokens;
      const T* x = static_cast<const T*>(p.q) + (there ? at * p.ld_q : 0) + (head * G + (there ? h : 0)) * D + 16 * t;
      float mul = 1.f;
      if constexpr (!std::is_same<T, __half>::value) {
        uint32_t top = 0;
        if (there)
#pragma unroll
          for (int i2 = 0; i2 < D / 64; ++i2) top = max(top, top_q16(x + 64 * i2));
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        mul = row_power(top);
      }
#pragma unroll
      for (int i2 = 0; i2 < D / 64; ++i2) {
        uint32_t w[8];
        load_q16(x + 64 * i2, there, mul, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          qb[j][i2 * 4 + k][0] = w[2 * k];
          qb[j][i2 * 4 + k][1] = w[2 * k + 1];
        }
      }
      const float f = p.scale * 1.4426950408889634f / mul;
      const int see = there ? static_cast<int>(max(static_cast<int64_t>(0), behind + i)) : 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qmul[j][e] = __shfl_sync(~0u, f, (2 * t + e) * 4);
        lim[j][e] = __shfl_sync(~0u, see, (2 * t + e) * 4);
        m[j][e] = mw[j][e] = kNone;
        l[j][e] = unit[j][e] = 0.f;
      }
    }

    float o[NQ][NV][4];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
#pragma unroll
      for (int i = 0; i < NV; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
    }

    float log_vs = -INFINITY;  // log2 of cur.vs, -infinity if that is 0 or no number
    for (int n = 0; n < mine; ++n) {
      const int stage = n % S;
      if ((n & 15) == 0) {
        if (n > 0) {
          cur = next;
          next = lookup(n + 16);
        }
        // not where it is looked up: the copies would wait for the scale
        log_vs = cur.vs > 0.f && cur.vs < INFINITY ? fminf(fmaxf(__log2f(cur.vs), kLeastLog2), kMostLog2) : -INFINITY;
      }
      const int src = 2 * (n & 15);
      const int id0 = __shfl_sync(~0u, cur.id, src), id1 = __shfl_sync(~0u, cur.id, src + 1);
      float ks[2], vs[2], lv[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = __shfl_sync(~0u, cur.ks, src + i);
        vs[i] = __shfl_sync(~0u, cur.vs, src + i);
        lv[i] = __shfl_sync(~0u, log_vs, src + i);
      }
      if (id1 < 0) lv[1] = lv[0];  // a half that is not there has no scores either
      else if (id0 < 0) lv[0] = lv[1];
      cp_async_wait<S - 1>();  // one group per step: this step's copies of this lane have landed,
      __syncwarp();            // and the other lanes'
      const uint8_t* kt = ring_ptr + stage * 2 * L::kHalf;
      const uint8_t* vt = kt + L::kHalf;

      float s[2][NQ][4];  // [16 keys][rows]: key g rows 2 t, 2 t + 1, key g + 8 rows 2 t, 2 t + 1
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          uint4 w[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int row = mt * 16 + u * 8 + prow;
            w[u] = *reinterpret_cast<const uint4*>(D == 128 ? kt + row * 128 + (((i * 4 + t) ^ (row & 7)) << 4)
                                                            : kt + row * 64 + ((t ^ ((row >> 1) & 3)) << 4));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t x = (k == 0 ? w[0].x : k == 1 ? w[0].y : k == 2 ? w[0].z : w[0].w) ^ 0x80808080u;
            const uint32_t y = (k == 0 ? w[1].x : k == 1 ? w[1].y : k == 2 ? w[1].z : w[1].w) ^ 0x80808080u;
            const uint32_t a[4] = {bytes_to_f16(x, 0x4140), bytes_to_f16(y, 0x4140), bytes_to_f16(x, 0x4342),
                                   bytes_to_f16(y, 0x4342)};
#pragma unroll
            for (int j = 0; j < NQ; ++j) mma_f16(s[mt][j], a, qb[j][i * 4 + k][0], qb[j][i * 4 + k][1]);
          }
        }
      }

      const int key0 = (first + n * W) * kStep;
      const bool edge = key0 + kStep > lim_first || id0 < 0 || id1 < 0;
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][j][e] *= qmul[j][e & 1] * ks[mt];
        }
      }
      if (edge) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + mt * 16 + (e >> 1) * 8 + prow >= lim[j][e & 1] || (mt == 0 ? id0 : id1) < 0)
                s[mt][j][e] = -INFINITY;
          }
        }
      }
      float mx[NQ][2], wx[NQ][2];  // maxima of this step, -infinity without a key
      bool up = false;
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float top[2] = {fmaxf(s[0][j][e], s[0][j][2 + e]), fmaxf(s[1][j][e], s[1][j][2 + e])};
          float x = fmaxf(top[0], top[1]);
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
          mx[j][e] = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
          wx[j][e] = mx[j][e] + lv[0];
          if (lv[0] != lv[1]) {  // two blocks, for the whole warp
            x = fmaxf(top[0] + lv[0], top[1] + lv[1]);
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
            wx[j][e] = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
          }
          up = up || mx[j][e] > m[j][e] + kMaxSlack || wx[j][e] > mw[j][e] + kMaxSlack;
        }
      }
      if (__any_sync(~0u, up)) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          float a[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mn = fmaxf(m[j][e], mx[j][e]);
            float wn = fmaxf(mw[j][e], wx[j][e]);
            if (wn > kNone) wn = fmaxf(wn, mn + kLeastLog2);  // the largest p may belong to a block without values
            l[j][e] *= exp2_approx(m[j][e] - mn);
            a[e] = exp2_approx(mw[j][e] - wn);
            unit[j][e] = wn > kNone ? exp2f(mn - wn) : 0.f;  // 0: the row's values so far are zeros
            m[j][e] = mn;
            mw[j][e] = wn;
          }
#pragma unroll
          for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][i][e] *= a[e & 1];
          }
        }
      }
      uint32_t pb[2][NQ][2], pr[2][NQ][2];  // P in f16, and what that rounding left out (kRest)
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        const float base[2] = {m[j][0] - kPScaleLog2, m[j][1] - kPScaleLog2};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w[2] = {vs[h] * unit[j][0], vs[h] * unit[j][1]};
          float pv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = exp2_approx(s[h][j][e] - base[e & 1]);
            l[j][e & 1] += x;
            pv[e] = x * w[e & 1];
          }
          if (edge) {  // 0 whatever the scale is
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + h * 16 + (e >> 1) * 8 + prow >= lim[j][e & 1] || (h == 0 ? id0 : id1) < 0) pv[e] = 0.f;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t high = pack2(pv[2 * e], pv[2 * e + 1], __half());
            pb[h][j][e] = transpose8x8(high);
            if constexpr (kRest) {
              float a, b;
              unpack2(high, a, b, __half());
              pr[h][j][e] = transpose8x8(pack2(pv[2 * e] - a, pv[2 * e + 1] - b, __half()));
            }
          }
        }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint4 vw[4];  // D = 64 uses the first two words
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = mt * 16 + (e >> 1) * 8 + ((e & 1) ? v1 : v0);
          if constexpr (D == 128) {
            vw[e] = *reinterpret_cast<const uint4*>(vt + row * 128 + ((g ^ (row & 7)) << 4));
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(vt + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8);
            vw[e] = make_uint4(w.x, w.y, 0, 0);
          }
        }
#pragma unroll
        for (int q4 = 0; q4 < D / 32; ++q4) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] = (q4 == 0 ? vw[e].x : q4 == 1 ? vw[e].y : q4 == 2 ? vw[e].z : vw[e].w) ^ 0x80808080u;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t lo = __byte_perm(x[0], x[1], u ? 0x7362 : 0x5140);
            const uint32_t hi = __byte_perm(x[2], x[3], u ? 0x7362 : 0x5140);
            const uint32_t a[4] = {bytes_to_f16(lo, 0x4140), bytes_to_f16(lo, 0x4342), bytes_to_f16(hi, 0x4140),
                                   bytes_to_f16(hi, 0x4342)};
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
              mma_f16(o[j][q4 * 2 + u], a, pb[mt][j][0], pb[mt][j][1]);
              if constexpr (kRest) mma_f16(o[j][q4 * 2 + u], a, pr[mt][j][0], pr[mt][j][1]);
            }
          }
        }
      }
      __syncwarp();  // every lane has its bytes: the stage may be filled again
      const int at = 2 * ((n + S) & 15);
      const bool same = ((n + S) >> 4) == (n >> 4), more = n + S < mine;
      const int ahead = same ? cur.id : next.id;
      const int a0 = __shfl_sync(~0u, ahead, at), a1 = __shfl_sync(~0u, ahead, at + 1);
      issue(n + S, more ? a0 : -1, more ? a1 : -1);
    }
    cp_async_wait<0>();

    // ---- the four warps' results become one
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[j][e] += __shfl_xor_sync(~0u, l[j][e], 4);
        l[j][e] += __shfl_xor_sync(~0u, l[j][e], 8);
        l[j][e] += __shfl_xor_sync(~0u, l[j][e], 16);
        if (g == 0) {
          part_m[warp][j * 8 + 2 * t + e] = m[j][e] == kNone ? -INFINITY : m[j][e];
          part_l[warp][j * 8 + 2 * t + e] = l[j][e] * exp2f(-kPScaleLog2);
        }
      }
    }
    __syncthreads();  // no ring is in use: partial outputs take their place
    float* parts = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = j * 8 + 2 * t + e;
        const float back = mw[j][e] == kNone ? 0.f : exp2f(mw[j][e] - m[j][e] - kPScaleLog2);
        if (row < rows) {
          float4* po = reinterpret_cast<float4*>(parts + (warp * ROWS + row) * D + g * (D / 8));
#pragma unroll
          for (int i = 0; i < NV; i += 2)
            po[i / 2] = make_float4(o[j][i][e] * back, o[j][i][2 + e] * back, o[j][i + 1][e] * back,
                                    o[j][i + 1][2 + e] * back);
        }
      }
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == rq.steps;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (s0 == 0 ? 1 : 0);
    for (int e = threadIdx.x; e < rows * D; e += kSplitThreads) {
      const int row = e / D, d = e % D;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, part_m[w][row]);
      float sum = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float a = top == -INFINITY ? 1.f : exp2_approx(part_m[w][row] - top);
        sum += a * part_l[w][row];
        acc += a * parts[(w * ROWS + row) * D + d];
      }
      if (whole) {
        const int64_t at = tok0 + (row0 + row) / G;
        if (at >= 0 && at < p.tokens)
          static_cast<T*>(p.out)[at * p.ld_out + (head * G + (row0 + row) % G) * D + d] =
              pack_one(sum == 0.f ? 0.f : acc / sum, T());
      } else {
        ws.o[(slot * ROWS + row) * D + d] = acc;
        if (d == 0) ws.ml[slot * ROWS + row] = make_float2(top, sum);
      }
    }
    if (!whole && s0 == 0 && threadIdx.x == 0) {
      // this item goes on in the next CTAs, up to the one that has its last step
      const int64_t begin = total * (blockIdx.x + 1) / gridDim.x;  // the first step that is not this CTA's
      const int64_t end = begin + rq.steps - s1;
      int n = 1;
      while (total * (blockIdx.x + n) / gridDim.x < end) ++n;
      ws.desc[blockIdx.x] = make_int4(r, head, tile, n);
    }
    __syncthreads();  // before the rings are filled again, or the next item's parts are written
    left -= s1 - s0;
    ++item;
    s0 = 0;
  }
}

// After the prompts' kernel of a mixed batch it waits for that one like any other.  (Starting on the SMs that the last
// prompt CTAs leave free took 71 us instead of 82 for 21 single tokens and 3 prompts of up to 511; but what the kernels
// before the prompts' wrote is promised behind the wait only, and another thread may launch something between the two.)
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(kSplitThreads, 3)
split_kernel(const __grid_constant__ Kv8AttentionParams p, SplitShape shape, SplitWs ws) {
  grid_dep_wait();
  grid_dep_launch();
  split_body<T, D, NQ>(p, shape, ws);
}

// Joins the pieces of the item that CTA blockIdx.x of split_kernel started.  D / 4 threads hold an output row; the
// groups of them take rows side by side when the pieces are few and the pieces of one row when they are many.
constexpr int kJoinThreads = 256;

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kJoinThreads)
join_kernel(const __grid_constant__ Kv8AttentionParams p, SplitShape shape, SplitWs ws) {
  constexpr int GROUPS = kJoinThreads / (D / 4);
  __shared__ float part[GROUPS][D], part_m[GROUPS], part_l[GROUPS];
  grid_dep_wait();
  grid_dep_launch();
  const int4 it = ws.desc[blockIdx.x];
  const int pieces = it.w;
  if (pieces <= 1) return;
  const int G = p.q_heads / p.cache.kv_heads;
  const Request q = request_of(p, it.x, shape.max_rows, ROWS);
  const int rows = min(ROWS, q.q_len * G - it.z * ROWS);
  const int64_t tok0 = p.q_start[it.x], c0 = blockIdx.x;
  int per_row = 1;  // groups that share a row
  while (per_row < GROUPS && per_row * 2 < pieces) per_row *= 2;
  const int at_once = GROUPS / per_row;
  const int group = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  const int part_of = group % per_row;
  for (int row0 = static_cast<int>(blockIdx.y) * at_once; row0 < rows; row0 += at_once * gridDim.y) {
    const int r = row0 + group / per_row;
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) {
#pragma unroll 4
      for (int i = part_of; i < pieces; i += per_row) {
        const int64_t slot = (i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)) * ROWS + r;
        const float2 ml = ws.ml[slot];
        const float4 v = *reinterpret_cast<const float4*>(ws.o + slot * D + d);
        if (ml.x == -INFINITY && ml.y == 0.f) continue;  // saw no key (its output may not even be written)
        const float mn = fmaxf(top, ml.x);
        const float a = mn == -INFINITY ? 1.f : exp2_approx(top - mn), b = mn == -INFINITY ? 1.f : exp2_approx(ml.x - mn);
        sum = sum * a + ml.y * b;
        acc = make_float4(acc.x * a + v.x * b, acc.y * a + v.y * b, acc.z * a + v.z * b, acc.w * a + v.w * b);
        top = mn;
      }
    }
    __syncthreads();  // the rows before have been read
    *reinterpret_cast<float4*>(&part[group][d]) = acc;
    if (d == 0) {
      part_m[group] = top;
      part_l[group] = sum;
    }
    __syncthreads();
    if (part_of == 0 && r < rows) {
      for (int i = 0; i < per_row; ++i) top = fmaxf(top, part_m[group + i]);
      sum = 0.f;
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = 0; i < per_row; ++i) {
        const float a = top == -INFINITY ? 1.f : exp2_approx(part_m[group + i] - top);
        const float4 v = *reinterpret_cast<const float4*>(&part[group + i][d]);
        sum += a * part_l[group + i];
        acc = make_float4(acc.x + a * v.x, acc.y + a * v.y, acc.z + a * v.z, acc.w + a * v.w);
      }
      const int row = it.z * ROWS + r;
      const int64_t at = tok0 + row / G;
      if (at >= 0 && at < p.tokens) {
        const bool none = sum == 0.f;
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * p.ld_out + (it.y * G + row % G) * D + d) =
            make_uint2(none ? 0u : pack2(acc.x / sum, acc.y / sum, T()), none ? 0u : pack2(acc.z / sum, acc.w / sum, T()));
      }
    }
  }
}

bool misaligned(const void* p, uintptr_t by) { return (reinterpret_cast<uintptr_t>(p) & (by - 1)) != 0; }

int stream_ctas() { return 3 * device_sm_count(); }

int64_t ws_bytes(int ctas, int dim) {
  return static_cast<int64_t>(ctas) * (2 * kMaxRows * (dim * 4 + 8) + 16);
}

template <typename T, int D, int NQ>
cudaError_t launch_split(const Kv8AttentionParams& p, const SplitShape& shape, dim3 grid, cudaStream_t stream,
                         const char** err) {
  SplitWs ws = {};
  if (shape.stream) {
    char* at = static_cast<char*>(p.workspace);
    ws.o = reinterpret_cast<float*>(at);
    at += static_cast<int64_t>(grid.x) * 2 * 8 * NQ * D * 4;
    ws.ml = reinterpret_cast<float2*>(at);
    at += static_cast<int64_t>(grid.x) * 2 * 8 * NQ * 8;
    ws.desc = reinterpret_cast<int4*>(at);
  }
  auto kern = split_kernel<T, D, NQ>;
  constexpr int smem = SplitSmem<D>::kDynamic;
  static std::atomic<uint64_t> ready{0};
  cudaError_t st = allow_smem(kern, smem, ready);
  if (st != cudaSuccess) return st;
  st = launch_dependent(kern, grid, dim3(kSplitThreads), smem, stream, p, shape, ws);
  if (st != cudaSuccess || !shape.stream) return st;
  return launch_dependent(join_kernel<T, D, 8 * NQ>, dim3(grid.x, 4), dim3(kJoinThreads), 0, stream, p, shape, ws);
}

template <typename T, int D>
cudaError_t launch_t(const Kv8AttentionParams& p, int max_rows, cudaStream_t stream, const char** err) {
  const int64_t rows = std::min(static_cast<int64_t>(p.max_q) * (p.q_heads / p.cache.kv_heads), static_cast<int64_t>(max_rows));
  const int nq = rows <= 8 ? 1 : 2;
  const int64_t row_tiles = (rows + 8 * nq - 1) / (8 * nq);
  const int64_t items = row_tiles * p.cache.kv_heads * p.requests;
  SplitShape shape;
  shape.max_rows = max_rows;
  shape.row_tiles = static_cast<int>(row_tiles);
  // one CTA per item: at most what kDirectMost keys take if the others have nothing to do meanwhile
  shape.stream = p.max_kv > kKv8DirectKeys && (p.max_kv > kDirectMost || items < 2 * stream_ctas()) ? 1 : 0;
  const dim3 grid = shape.stream ? dim3(static_cast<unsigned>(stream_ctas()))
                                 : dim3(static_cast<unsigned>(shape.row_tiles * p.cache.kv_heads),
                                        static_cast<unsigned>(p.requests));
  return nq == 1 ? launch_split<T, D, 1>(p, shape, grid, stream, err) : launch_split<T, D, 2>(p, shape, grid, stream, err);
}

}  // namespace

int64_t kv8_attention_workspace_bytes(const Kv8AttentionParams& p) {
  if (p.max_kv <= kKv8DirectKeys || kv8_cache_problem(p.cache) || p.q_heads < p.cache.kv_heads || p.q_heads > 65535 ||
      p.tokens <= 0 || p.tokens > INT32_MAX)
    return 0;
  const bool many = static_cast<int64_t>(p.max_q) * (p.q_heads / p.cache.kv_heads) > kSplitRows;
  return (!many || p.requests > 1 ? ws_bytes(stream_ctas(), p.cache.dim) : 0) + (many ? kv8_prefill_workspace_bytes(p) : 0);
}

cudaError_t kv8_attention_launch(const Kv8AttentionParams& p, cudaStream_t stream, const char** err) {
  *err = kv8_cache_problem(p.cache);
  const int64_t row = static_cast<int64_t>(p.q_heads) * p.cache.dim;
  if (*err) return cudaErrorInvalidValue;
  if (p.type != kKvF16 && p.type != kKvBF16) *err = "element type must be f16 or bf16";
  else if (p.q_heads <= 0 || p.q_heads % p.cache.kv_heads != 0 || p.q_heads > 65535)
    *err = "query heads must be a multiple of the kv heads";
  else if (p.tokens < 0 || p.tokens > INT32_MAX || p.requests < 0 || p.requests > 65535 || p.table_width < 0 ||
           p.max_q < 0 || p.max_kv < 0)
    *err = "sizes out of range";
  else if (static_cast<int64_t>(p.table_width) * p.cache.block_size > (1 << 30))
    *err = "positions are 32-bit: the table is too wide";
  if (*err) return cudaErrorInvalidValue;
  if (p.tokens == 0 || p.requests == 0 || p.max_q == 0) return cudaSuccess;
  if (!p.q || !p.out || (!p.table && p.table_width > 0) || !p.q_start || !p.q_lens || !p.kv_lens)
    *err = "null operand";
  else if (p.ld_q < row || p.ld_out < row || p.ld_q % 8 != 0 || p.ld_out % 8 != 0 || misaligned(p.q, 16) ||
           misaligned(p.out, 16))
    *err = "rows of q and out must hold all heads, 16-byte aligned";
  else if (!(p.scale > 0.f))
    *err = "the score scale must be positive";
  if (*err) return cudaErrorInvalidValue;
  // Which requests go where is decided on the device, from q_lens; the host knows the bound.
  const int64_t rows = static_cast<int64_t>(p.max_q) * (p.q_heads / p.cache.kv_heads);
  const bool many = rows > kSplitRows, few = !many || p.requests > 1;
  const int64_t need = kv8_attention_workspace_bytes(p);
  if (need > 0 && (!p.workspace || misaligned(p.workspace, 16) || p.workspace_bytes < need))
    *err = "the workspace is too small or not 16-byte aligned";
  if (p.cache.num_blocks == 0) *err = "a cache without blocks";
  if (*err) return cudaErrorInvalidValue;
  // the prompts' shares lie behind the pieces of the few rows
  void* shares = few && need > 0 ? static_cast<char*>(p.workspace) + ws_bytes(stream_ctas(), p.cache.dim) : p.workspace;
  cudaError_t st = cudaSuccess;
  if (many) st = kv8_prefill_launch(p, few ? kSplitRowsMixed : 0, shares, stream, err);
  if (st == cudaSuccess && few) {
    const int most = many ? kSplitRowsMixed : kSplitRows;
    const bool f16 = p.type == kKvF16;
    if (p.cache.dim == 128)
      st = f16 ? launch_t<__half, 128>(p, most, stream, err) : launch_t<__nv_bfloat16, 128>(p, most, stream, err);
    else
      st = f16 ? launch_t<__half, 64>(p, most, stream, err) : launch_t<__nv_bfloat16, 64>(p, most, stream, err);
  }
  if (st == cudaSuccess && many) st = kv8_prefill_join_launch(p, few ? kSplitRowsMixed : 0, shares, stream);
  return st;
}

}  // namespace disc_b200
