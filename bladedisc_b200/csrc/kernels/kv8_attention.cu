// Attention over the 8-bit paged cache:
//   s_ij = scale * k_scale[block(j)] * (q_i . k_j),   j <= kv_len - q_len + i
//   o_i  = sum_j softmax(s_i)_j * v_scale[block(j)] * v_j,   0 where row i sees no key.
#include "kv8.h"

#include <type_traits>

#include "device_info.h"
#include "kv8_types.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.h"

namespace disc_b200 {

__device__ int g_kv8_status = 0;

namespace {

// ------------------------------------------------------------------------------------------------ few rows
// Up to a few dozen query rows per request and kv head: the cache is read once and its bytes are what bounds the
// kernel, closely followed by the instructions that turn levels into f16.
//
// An item is a request, a kv head and 16 query rows (query heads of that kv head, tokens of that request); its work
// is steps of 32 keys.  All steps of all items are laid end to end and cut into equal shares, one per CTA, three CTAs
// per SM: ragged lengths balance to one step.  A share that ends inside an item leaves its partial maximum, sum and
// output in the workspace, and a second small kernel joins them.  Short caches (max_kv <= kDirectKeys) take one CTA
// per item and need neither.
//
// Inside a CTA a warp runs by itself: it fetches its steps with TMA into its own ring, multiplies with mma.sync
// m16n8k16, keeps running maximum, sum and output in registers and meets the others at the end of the item.
//
//   S = Q K^T  the head dimension is permuted alike in Q and K so that a lane's B fragments are the bytes of 16-byte
//              loads; levels become f16 exactly (byte b as 0x6400 | b + 128 is 1152 + b, one subtraction).
//   O += P V   a lane's B fragments pair bytes of two keys: two byte permutes, again exact in f16.
// Query rows in bf16 are scaled by a power of two per row to f16 (exact but for values 2^-24 of the row's largest).
// P goes to f16 with 2^13 of head room so that a probability keeps its 11 bits down to 2^-27 of the largest; the
// value scale is multiplied in relative to a running reference that O is kept in units of.
// The 128-byte (64-byte for dim 64) swizzle of the TMA boxes and the key order perm(n) = n ^ ((n & 1) << 2) make the
// 16-byte shared-memory reads free of bank conflicts.
constexpr int kStep = 32;         // keys per step of a warp
constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = kSplitWarps * 32;
constexpr int kDirectKeys = 512;  // caches up to this long are not cut
constexpr float kPScaleLog2 = 13.f;
constexpr float kRefSlack = 4.f;  // a value scale may exceed the reference by this much before O is rescaled
constexpr float kRef0 = 1e-30f;

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Bytes b (as b + 128) `sel` picks two of them -> two f16 with the values b.
__device__ __forceinline__ uint32_t bytes_to_f16(uint32_t biased, uint32_t sel) {
  const uint32_t w = __byte_perm(biased, 0x64646464u, sel);
  const uint32_t c = 0x64806480u;  // 1152
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
// Largest magnitude of sixteen values, as its bits.
__device__ __forceinline__ uint32_t top_q16(const __nv_bfloat16* p) {
  float f[16];
  load8(p, f);
  load8(p + 8, f + 8);
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) t = max(t, __float_as_uint(f[i]) & 0x7fffffffu);
  return t;
}
// 2^n that brings a row with this largest magnitude to [2^13, 2^14); n stays within what a float holds.
__device__ __forceinline__ float row_power(uint32_t top) {
  const int n = min(max(13 - (static_cast<int>(top >> 23) - 127), -120), 120);
  return __uint_as_float(static_cast<uint32_t>(n + 127) << 23);
}

// What is left of a share that ends inside an item: a maximum, a sum and an output per row.
struct SplitWs {
  float* o;      // [2 * ctas][16][dim]: slot 2 c for a piece that does not start its item, 2 c + 1 for one that does
  float2* ml;    // [2 * ctas][16]
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
  static constexpr int kParts = kSplitWarps * 16 * D * 4;  // O of every warp, in the place of the rings
  static constexpr int kDynamic = (kRing > kParts ? kRing : kParts) + 1024;
};

// Query rows (tokens x heads of a group) and steps of one request; no rows if the request is not for this kernel.
struct Request {
  int q_asked, q_len, kv_len, tiles, steps;
};
__device__ __forceinline__ Request request_of(const Kv8AttentionParams& p, int r, int max_rows) {
  Request q;
  const int G = p.q_heads / p.cache.kv_heads;
  q.q_asked = max(p.q_lens[r], 0);
  q.q_len = min(q.q_asked, p.max_q);
  q.kv_len = min(max(p.kv_lens[r], 0), p.table_width * p.cache.block_size);
  const int64_t rows = static_cast<int64_t>(q.q_asked) * G <= max_rows ? static_cast<int64_t>(q.q_len) * G : 0;
  q.tiles = static_cast<int>((rows + 15) / 16);
  q.steps = max(1, (q.kv_len + kStep - 1) / kStep);
  return q;
}

template <typename T, int D, bool HI>
__global__ void __launch_bounds__(kSplitThreads, 3)
split_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
             const __grid_constant__ Kv8AttentionParams p, SplitShape shape, SplitWs ws) {
  using L = SplitSmem<D>;
  constexpr int W = kSplitWarps, S = L::kStages;
  constexpr int KQ = D / 16;  // k steps of the first product
  constexpr int NV = D / 8;   // n tiles of the second
  constexpr int E = HI ? 2 : 1;  // rows per lane: g, and g + 8 when there may be more than eight
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t bars[W * S];
  __shared__ float part_m[W][16], part_l[W][16];
  __shared__ long long sums[W];
  __shared__ int found[2];
  __shared__ long long found_at;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;

  const Kv8Cache& c = p.cache;
  const int bs = c.block_size, G = p.q_heads / c.kv_heads, KH = c.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  if (threadIdx.x == 0) {
    abort_word = 0;
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (lane < S) mbar_init(smem_u32(&bars[warp * S + lane]), 1);
  fence_mbar_init();
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();

  // ---- which steps are this CTA's: `left` steps from step `s0` of item `item` of request r on
  int r;
  int64_t left, item, s0, total = 0;
  if (!shape.stream) {
    r = blockIdx.y;
    const Request q = request_of(p, r, shape.max_rows);
    const int tile = blockIdx.x % shape.row_tiles;
    if (tile >= q.tiles) return;
    item = static_cast<int64_t>(blockIdx.x / shape.row_tiles) * q.tiles + tile;
    s0 = 0;
    left = q.steps;
  } else {
    const int per = (p.requests + kSplitThreads - 1) / kSplitThreads;
    const int r0 = min(p.requests, static_cast<int>(threadIdx.x) * per), r1 = min(p.requests, r0 + per);
    int64_t mine = 0;
    for (int i = r0; i < r1; ++i) {
      const Request q = request_of(p, i, shape.max_rows);
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
        const Request q = request_of(p, i, shape.max_rows);
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
      if (threadIdx.x < 16) ws.ml[static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x] = make_float2(-INFINITY, 0.f);
      return;
    }
    r = found[0];
    const Request q = request_of(p, r, shape.max_rows);
    item = found_at / q.steps;
    s0 = found_at % q.steps;
  }
  Request rq = request_of(p, r, shape.max_rows);

  const uint32_t ring = smem_u32(smem) + warp * (S * 2 * L::kHalf);
  const uint8_t* ring_ptr = smem + warp * (S * 2 * L::kHalf);
  const uint32_t bar0 = smem_u32(&bars[warp * S]);
  const int prow = g ^ ((g & 1) << 2);         // key of n = g in a group of eight
  const int v0 = 2 * t, v1 = (2 * t + 1) ^ 4;  // keys of this lane's columns
  uint32_t waits = 0;                          // steps that this warp's ring has delivered
  bool ok = true;

  while (left > 0) {
    while (item >= static_cast<int64_t>(rq.tiles) * KH) {  // on to the next request with rows
      if (++r >= p.requests) return;  // not with lengths that stay as they are during the call
      item = 0;
      rq = request_of(p, r, shape.max_rows);
    }
    const int head = static_cast<int>(item / rq.tiles), tile = static_cast<int>(item % rq.tiles);
    const int s1 = static_cast<int>(min(static_cast<int64_t>(rq.steps), s0 + left));
    const int64_t row0 = static_cast<int64_t>(tile) * 16;
    const int rows = static_cast<int>(min(static_cast<int64_t>(16), static_cast<int64_t>(rq.q_len) * G - row0));
    const int64_t tok0 = p.q_start[r];
    const int64_t behind = static_cast<int64_t>(rq.kv_len) - rq.q_asked + 1;
    // keys that the first row of the tile sees, and the last one
    const int lim_first = static_cast<int>(max(static_cast<int64_t>(0), behind + row0 / G));
    const int keys = static_cast<int>(max(static_cast<int64_t>(0), behind + (row0 + rows - 1) / G));

    // Q fragments of rows g and g + 8
    uint32_t qa[KQ][4];
    float qmul[E];
    int lim[E];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (e >= E) {
#pragma unroll
        for (int j = 0; j < KQ; ++j) qa[j][1] = qa[j][3] = 0;
        continue;
      }
      const int row = g + 8 * e;
      const int64_t i = (row0 + row) / G, h = (row0 + row) % G;
      const int64_t at = tok0 + i;
      const bool there = row < rows && at >= 0 && at < p.tokens;
      lim[e] = there ? static_cast<int>(max(static_cast<int64_t>(0), behind + i)) : 0;
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
        for (int j = 0; j < 4; ++j) {
          qa[i2 * 4 + j][e] = w[2 * j];
          qa[i2 * 4 + j][2 + e] = w[2 * j + 1];
        }
      }
      qmul[e] = p.scale * 1.4426950408889634f / mul;
    }

    float o[NV][4];
#pragma unroll
    for (int j = 0; j < NV; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m[E], l[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      m[e] = -INFINITY;
      l[e] = 0.f;
    }
    float ref = kRef0, inv_ref = 1.f / kRef0;

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
    auto issue = [&](int n, int stage, int id0, int id1) {  // lane 0
      const uint32_t bar = bar0 + 8 * stage, kt = ring + stage * 2 * L::kHalf;
      const int off = ((first + n * W) * kStep) & (bs - 1);
      if (bs >= kStep) {  // both halves lie in one block
        if (id0 < 0) {
          mbar_arrive(bar);
          return;
        }
        mbar_arrive_expect_tx(bar, 2 * L::kHalf);
        tma_load_3d(kt, &tk, bar, 0, off, id0 * KH + head);
        tma_load_3d(kt + L::kHalf, &tv, bar, 0, off, id0 * KH + head);
      } else {
        const int n_there = (id0 >= 0) + (id1 >= 0);
        if (n_there == 0) {
          mbar_arrive(bar);
          return;
        }
        mbar_arrive_expect_tx(bar, n_there * L::kHalf);
        if (id0 >= 0) {
          tma_load_3d(kt, &tk, bar, 0, 0, id0 * KH + head);
          tma_load_3d(kt + L::kHalf, &tv, bar, 0, 0, id0 * KH + head);
        }
        if (id1 >= 0) {
          tma_load_3d(kt + L::kHalf / 2, &tk, bar, 0, 0, id1 * KH + head);
          tma_load_3d(kt + L::kHalf + L::kHalf / 2, &tv, bar, 0, 0, id1 * KH + head);
        }
      }
    };

    cur = lookup(0);
#pragma unroll
    for (int n = 0; n < S; ++n) {
      const int id0 = __shfl_sync(~0u, cur.id, 2 * n), id1 = __shfl_sync(~0u, cur.id, 2 * n + 1);
      if (ok && n < mine && lane == 0) issue(n, (waits + n) % S, id0, id1);
    }
    next = lookup(16);

    for (int n = 0; n < mine && ok; ++n, ++waits) {
      const int stage = waits % S;
      if ((n & 15) == 0 && n > 0) {
        cur = next;
        next = lookup(n + 16);
      }
      const int src = 2 * (n & 15);
      const int id0 = __shfl_sync(~0u, cur.id, src), id1 = __shfl_sync(~0u, cur.id, src + 1);
      float ks[2], vs[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = __shfl_sync(~0u, cur.ks, src + i);
        vs[i] = __shfl_sync(~0u, cur.vs, src + i);
      }
      ok = mbar_wait(bar0 + 8 * stage, (waits / S) & 1, abort_flag, &g_kv8_status, 41);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      const uint8_t* kt = ring_ptr + stage * 2 * L::kHalf;
      const uint8_t* vt = kt + L::kHalf;

      float s[4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
        const int row = nt * 8 + prow;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint4 w = *reinterpret_cast<const uint4*>(
              D == 128 ? kt + row * 128 + (((i * 4 + t) ^ (row & 7)) << 4) : kt + row * 64 + ((t ^ ((row >> 1) & 3)) << 4));
          const uint32_t x[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_f16(s[nt], qa[i * 4 + j], bytes_to_f16(x[j], 0x4140), bytes_to_f16(x[j], 0x4342));
        }
      }

      const int key0 = (first + n * W) * kStep;
      const bool edge = key0 + kStep > lim_first || id0 < 0 || id1 < 0;
      float mn[E];
      bool up = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float mx = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
          const float f = qmul[e] * ks[nt >> 1];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float& x = s[nt][2 * e + j];
            x *= f;
            if (edge && (key0 + nt * 8 + (j ? v1 : v0) >= lim[e] || (nt < 2 ? id0 : id1) < 0)) x = -INFINITY;
            mx = fmaxf(mx, x);
          }
        }
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
        mn[e] = fmaxf(m[e], mx);
        up = up || mn[e] > m[e];
      }
      float vtop = vs[0] < INFINITY ? vs[0] : 0.f;
      vtop = vs[1] < INFINITY ? fmaxf(vtop, vs[1]) : vtop;
      const bool grow = vtop > kRefSlack * ref;
      if (__any_sync(~0u, up) || grow) {
        float down = 1.f;
        if (grow) {
          down = ref / vtop;
          ref = vtop;
          inv_ref = 1.f / vtop;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float a = mn[e] == -INFINITY ? 1.f : exp2_approx(m[e] - mn[e]);
          m[e] = mn[e];
          l[e] *= a;
          a *= down;
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            o[j][2 * e] *= a;
            o[j][2 * e + 1] *= a;
          }
        }
      }
      uint32_t pa[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (e >= E) {
          pa[0][1] = pa[0][3] = pa[1][1] = pa[1][3] = 0;
          continue;
        }
        const float base = (m[e] == -INFINITY ? 0.f : m[e]) - kPScaleLog2;
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
          const float w = vs[nt >> 1] * inv_ref;
          float pv[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float x = exp2_approx(s[nt][2 * e + j] - base);
            l[e] += x;
            pv[j] = x * w;
            // whatever the scale is
            if (edge && (key0 + nt * 8 + (j ? v1 : v0) >= lim[e] || (nt < 2 ? id0 : id1) < 0)) pv[j] = 0.f;
          }
          pa[nt >> 1][(nt & 1) * 2 + e] = pack2(pv[0], pv[1], __half());
        }
      }
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        uint4 vw[4];  // D = 64 uses the first two words
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = h2 * 16 + (e >> 1) * 8 + ((e & 1) ? v1 : v0);
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
          const uint32_t a01 = __byte_perm(x[0], x[1], 0x5140), a23 = __byte_perm(x[0], x[1], 0x7362);
          const uint32_t b01 = __byte_perm(x[2], x[3], 0x5140), b23 = __byte_perm(x[2], x[3], 0x7362);
          mma_f16(o[q4 * 4 + 0], pa[h2], bytes_to_f16(a01, 0x4140), bytes_to_f16(b01, 0x4140));
          mma_f16(o[q4 * 4 + 1], pa[h2], bytes_to_f16(a01, 0x4342), bytes_to_f16(b01, 0x4342));
          mma_f16(o[q4 * 4 + 2], pa[h2], bytes_to_f16(a23, 0x4140), bytes_to_f16(b23, 0x4140));
          mma_f16(o[q4 * 4 + 3], pa[h2], bytes_to_f16(a23, 0x4342), bytes_to_f16(b23, 0x4342));
        }
      }
      __syncwarp();  // every lane has its bytes: the stage may be filled again
      if (n + S < mine) {
        const int at = 2 * ((n + S) & 15);
        const int a0 = __shfl_sync(~0u, cur.id, at), a1 = __shfl_sync(~0u, cur.id, at + 1);
        const int b0 = __shfl_sync(~0u, next.id, at), b1 = __shfl_sync(~0u, next.id, at + 1);
        const bool same = ((n + S) >> 4) == (n >> 4);
        if (lane == 0) issue(n + S, stage, same ? a0 : b0, same ? a1 : b1);
      }
    }
    if (!ok) {  // let copies in flight land before the shared memory is used or given back
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    }

    // ---- the four warps' results become one
#pragma unroll
    for (int e = 0; e < E; ++e) {
      l[e] += __shfl_xor_sync(~0u, l[e], 1);
      l[e] += __shfl_xor_sync(~0u, l[e], 2);
      if (t == 0) {
        part_m[warp][g + 8 * e] = m[e];
        part_l[warp][g + 8 * e] = l[e] * exp2f(-kPScaleLog2);
      }
    }
    __syncthreads();  // no ring is in use: partial outputs take their place
    float* parts = reinterpret_cast<float*>(smem);
    const float unit = ref * exp2f(-kPScaleLog2);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (g + 8 * e < rows) {
        float* po = parts + (warp * 16 + g + 8 * e) * D;
#pragma unroll
        for (int j = 0; j < NV; j += 4) {
          *reinterpret_cast<float4*>(po + 2 * t * NV + j) =
              make_float4(o[j][2 * e] * unit, o[j + 1][2 * e] * unit, o[j + 2][2 * e] * unit, o[j + 3][2 * e] * unit);
          *reinterpret_cast<float4*>(po + (2 * t + 1) * NV + j) =
              make_float4(o[j][2 * e + 1] * unit, o[j + 1][2 * e + 1] * unit, o[j + 2][2 * e + 1] * unit,
                          o[j + 3][2 * e + 1] * unit);
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
        acc += a * parts[(w * 16 + row) * D + d];
      }
      if (whole) {
        const int64_t at = tok0 + (row0 + row) / G;
        if (at >= 0 && at < p.tokens)
          static_cast<T*>(p.out)[at * p.ld_out + (head * G + (row0 + row) % G) * D + d] =
              pack_one(sum == 0.f ? 0.f : acc / sum, T());
      } else {
        ws.o[(slot * 16 + row) * D + d] = acc;
        if (d == 0) ws.ml[slot * 16 + row] = make_float2(top, sum);
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

// Joins the pieces of the item that CTA blockIdx.x of split_kernel started: one block per row.
template <typename T, int D>
__global__ void __launch_bounds__(D) join_kernel(const __grid_constant__ Kv8AttentionParams p, SplitShape shape, SplitWs ws) {
  grid_dep_wait();
  grid_dep_launch();
  const int4 it = ws.desc[blockIdx.x];
  if (it.w <= 1) return;
  const int G = p.q_heads / p.cache.kv_heads;
  const Request q = request_of(p, it.x, shape.max_rows);
  const int64_t row = static_cast<int64_t>(it.z) * 16 + blockIdx.y;
  if (row >= static_cast<int64_t>(q.q_len) * G) return;
  const int64_t at = p.q_start[it.x] + row / G;
  if (at < 0 || at >= p.tokens) return;
  const int64_t c0 = blockIdx.x;
  float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll 4
  for (int i = 0; i < it.w; ++i) {
    const int64_t slot = ((i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)) * 16) + blockIdx.y;
    const float2 ml = ws.ml[slot];
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // saw no key (its output may not even be written)
    const float v = ws.o[slot * D + threadIdx.x];
    const float mn = fmaxf(top, ml.x);
    const float a = mn == -INFINITY ? 1.f : exp2_approx(top - mn), b = mn == -INFINITY ? 1.f : exp2_approx(ml.x - mn);
    sum = sum * a + ml.y * b;
    acc = acc * a + v * b;
    top = mn;
  }
  static_cast<T*>(p.out)[at * p.ld_out + (it.y * G + row % G) * D + threadIdx.x] =
      pack_one(sum == 0.f ? 0.f : acc / sum, T());
}

bool misaligned(const void* p, uintptr_t by) { return (reinterpret_cast<uintptr_t>(p) & (by - 1)) != 0; }

// One box is `rows` tokens of one block and head.
bool make_map(CUtensorMap* tm, const int8_t* base, const Kv8Cache& c, int rows) {
  EncodeTiledFn fn = tensor_map_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(c.dim), static_cast<cuuint64_t>(c.block_size),
                        static_cast<cuuint64_t>(c.num_blocks) * c.kv_heads};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(c.dim), static_cast<cuuint64_t>(c.dim) * c.block_size};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(c.dim), static_cast<cuuint32_t>(rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, c.dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int stream_ctas() { return 3 * device_sm_count(); }

int64_t ws_bytes(int ctas, int dim) {
  return static_cast<int64_t>(ctas) * (2 * 16 * (static_cast<int64_t>(dim) * 4 + 8) + 16);
}

bool wants_stream(const Kv8AttentionParams& p) { return p.max_kv > kDirectKeys; }

template <typename T, int D, bool HI>
cudaError_t launch_split(const Kv8AttentionParams& p, const SplitShape& shape, dim3 grid, cudaStream_t stream,
                         const char** err) {
  CUtensorMap tk, tv;
  const int box = p.cache.block_size < kStep ? p.cache.block_size : kStep;
  if (!make_map(&tk, p.cache.k, p.cache, box) || !make_map(&tv, p.cache.v, p.cache, box)) {
    *err = "cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  SplitWs ws = {};
  if (shape.stream) {
    char* at = static_cast<char*>(p.workspace);
    ws.o = reinterpret_cast<float*>(at);
    at += static_cast<int64_t>(grid.x) * 2 * 16 * D * 4;
    ws.ml = reinterpret_cast<float2*>(at);
    at += static_cast<int64_t>(grid.x) * 2 * 16 * 8;
    ws.desc = reinterpret_cast<int4*>(at);
  }
  auto kern = split_kernel<T, D, HI>;
  constexpr int smem = SplitSmem<D>::kDynamic;
  cudaError_t st = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (st != cudaSuccess) return st;
  st = launch_dependent(kern, grid, dim3(kSplitThreads), smem, stream, tk, tv, p, shape, ws);
  if (st != cudaSuccess || !shape.stream) return st;
  return launch_dependent(join_kernel<T, D>, dim3(grid.x, HI ? 16 : 8), dim3(D), 0, stream, p, shape, ws);
}

template <typename T, int D>
cudaError_t launch_t(const Kv8AttentionParams& p, cudaStream_t stream, const char** err) {
  const int64_t rows = static_cast<int64_t>(p.max_q) * (p.q_heads / p.cache.kv_heads);
  SplitShape shape;
  shape.max_rows = INT32_MAX;
  shape.stream = wants_stream(p) ? 1 : 0;
  const int64_t tiles = (rows + 15) / 16;
  if (tiles * p.cache.kv_heads > INT32_MAX) {
    *err = "too many query rows";
    return cudaErrorInvalidValue;
  }
  shape.row_tiles = static_cast<int>(tiles);
  const dim3 grid = shape.stream ? dim3(static_cast<unsigned>(stream_ctas()))
                                 : dim3(static_cast<unsigned>(tiles * p.cache.kv_heads), static_cast<unsigned>(p.requests));
  return rows > 8 ? launch_split<T, D, true>(p, shape, grid, stream, err)
                  : launch_split<T, D, false>(p, shape, grid, stream, err);
}

}  // namespace

int64_t kv8_attention_workspace_bytes(int32_t dim, int64_t max_kv) {
  return max_kv > kDirectKeys ? ws_bytes(stream_ctas(), dim) : 0;
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
  else if (static_cast<int64_t>(p.table_width) * p.cache.block_size > INT32_MAX)
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
  if (wants_stream(p) && (!p.workspace || misaligned(p.workspace, 16) || p.workspace_bytes < ws_bytes(stream_ctas(), p.cache.dim)))
    *err = "the workspace is too small or not 16-byte aligned";
  if (p.table_width == 0) {  // no keys at all, but the kernel's tensor maps want a cache
    if (p.cache.num_blocks == 0) *err = "a cache without blocks";
  }
  if (*err) return cudaErrorInvalidValue;
  if (p.cache.dim == 128)
    return p.type == kKvF16 ? launch_t<__half, 128>(p, stream, err) : launch_t<__nv_bfloat16, 128>(p, stream, err);
  return p.type == kKvF16 ? launch_t<__half, 64>(p, stream, err) : launch_t<__nv_bfloat16, 64>(p, stream, err);
}

int kv8_status_fetch_and_clear() {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, g_kv8_status, sizeof(int)) != cudaSuccess) return -1;
  if (h != 0) {
    int z = 0;
    cudaMemcpyToSymbol(g_kv8_status, &z, sizeof(int));
  }
  return h;
}

}  // namespace disc_b200
