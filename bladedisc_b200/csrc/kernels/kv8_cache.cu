// Append to the 8-bit cache and reading blocks back.
//
// A block of tokens and a head share one scale s = max|x| / 127 over the tokens stored since its first one (those that
// a trim took back too), levels are rne(x / s).  When new tokens raise the maximum of a block that already holds tokens, those are moved to the
// new scale: level' = rne(level * (s_old / s)); the error that adds is at most half a level each time the maximum
// grows.  Keys are rotated (pairs (i, i + dim / 2)) in fp32 and quantized without a rounding in between.
//
// Prompts: 9815 tokens with 32 query and 8 + 8 key / value heads of 128 values in bf16 move 225 MB in 54 us (0.63 of the
// measured copy rate), issue slots half busy: memory latency at 35 % of the warps, and every run is rotated twice.  Reading
// 315 blocks back moves 65 MB in 12.4 us (0.80).  Decode steps are latency: 64 tokens with 32 + 32 + 32 heads 7.4 us.
#include "kv8.h"

#include "device_info.h"
#include "kv8_types.cuh"
#include "sm100_ptx.cuh"

namespace disc_b200 {
namespace {

constexpr int kThreads = 128;

// (lo, hi) -> (lo c - hi s, hi c + lo s), each product and sum rounded once.
__device__ __forceinline__ void rotate8(float* lo, float* hi, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = lo[i], b = hi[i];
    lo[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
    hi[i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
  }
}

__device__ __forceinline__ void load_f8(const float* p, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// A level as the low byte of v + 1.5 2^23: rounded half to even, no conversion instruction.
__device__ __forceinline__ uint32_t level_bits(float v) {
  return __float_as_uint(fminf(fmaxf(v, -127.f), 127.f) + 12582912.f);
}
__device__ __forceinline__ uint32_t pack_bytes(const uint32_t* b) {
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}
// Levels of four values at scale s, inv = rn(1 / s): the quotient corrected by its own remainder (Markstein) is the
// correctly rounded x / s for normal operands, so that the level is that of the division at a third of its
// instructions.  inv = 0: 1 / s is not a normal number.
__device__ __forceinline__ uint32_t pack_levels(const float* x, float s, float inv) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = x[i] * inv;
    b[i] = level_bits(inv > 0.f ? fmaf(fmaf(-q, s, x[i]), inv, q) : __fdiv_rn(x[i], s));
  }
  return pack_bytes(b);
}

// Tokens of a run: the consecutive tokens whose slots follow one another inside one block.
constexpr int kMaxSegment = 128;  // tokens per block of threads, and the longest run
constexpr int kPasses = 4;        // passes over a run whose loads are in flight together
constexpr int kQPasses = 4;       // (token, query head) pairs per thread

// The first kv_blocks CTAs take a segment of `seg` consecutive tokens and four key / value heads each, a warp per head:
// every run whose first token lies in the segment, once for the maximum and once for the levels, eight values of each
// half of the head per lane; the second read comes from the caches (keeping a run in registers instead took 128 of
// them and was slower: 79 against 72 us for 9815 tokens).  Nothing is shared between warps but the slots.  The other CTAs rotate q, a thread
// for eight values of each half of kQPasses heads.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 6) append_kernel(const __grid_constant__ Kv8AppendParams p, int seg, int kv_blocks) {
  constexpr int half = D / 2;
  constexpr int kLanes = D / 16;          // lanes per token: eight values of each half of the head
  constexpr int kTokens = 32 / kLanes;    // tokens per pass of a warp
  const Kv8Cache& c = p.cache;
  const int bs = c.block_size;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk = lane % kLanes;
  const T* qkv = static_cast<const T*>(p.qkv);
  const int kv_groups = (2 * c.kv_heads + 3) / 4;
  grid_dep_wait();
  grid_dep_launch();

  if (static_cast<int>(blockIdx.x) >= kv_blocks) {
    constexpr int kPairs = kThreads / kLanes;
    T* out = static_cast<T*>(p.q_out);
    const uint32_t n = static_cast<uint32_t>(p.tokens * p.q_heads), q_heads = p.q_heads;
    const uint32_t i0 = (blockIdx.x - kv_blocks) * (kPairs * kQPasses) + threadIdx.x / kLanes;
    uint4 w[kQPasses][2];
    int pos[kQPasses];
#pragma unroll
    for (int e = 0; e < kQPasses; ++e) {
      const uint32_t i = i0 + e * kPairs;
      if (i < n) {
        const uint32_t t = i / q_heads, h = i - t * q_heads;
        const T* x = qkv + t * p.ld_qkv + h * D + chunk * 8;
        w[e][0] = *reinterpret_cast<const uint4*>(x);
        w[e][1] = *reinterpret_cast<const uint4*>(x + half);
        pos[e] = min(max(p.positions[t], 0), p.table_rows - 1);
      }
    }
#pragma unroll
    for (int e = 0; e < kQPasses; ++e) {
      const uint32_t i = i0 + e * kPairs;
      if (i < n) {
        float cs[8], sn[8], lo[8], hi[8];
        load_f8(p.cos_table + static_cast<int64_t>(pos[e]) * half + chunk * 8, cs);
        load_f8(p.sin_table + static_cast<int64_t>(pos[e]) * half + chunk * 8, sn);
        unpack8(w[e][0], lo, T());
        unpack8(w[e][1], hi, T());
        rotate8(lo, hi, cs, sn);
        T* o = out + static_cast<int64_t>(i) * D + chunk * 8;
        store8(o, lo);
        store8(o + half, hi);
      }
    }
    return;
  }
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / kv_groups) * seg;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(seg), p.tokens - t0));

  // slots of the segment, the token before it and the block's worth behind it; -2: no such token
  __shared__ int32_t slot_of[1 + 2 * kMaxSegment], pos_of[1 + 2 * kMaxSegment];
  for (int i = threadIdx.x; i < 1 + tokens + bs; i += kThreads) {
    const int64_t t = t0 - 1 + i;
    const bool there = t >= 0 && t < p.tokens;
    slot_of[i] = there ? p.slots[t] : -2;
    if (p.cos_table) pos_of[i] = there ? min(max(p.positions[t], 0), p.table_rows - 1) : 0;
  }
  __syncthreads();
  const int y = blockIdx.x % kv_groups * 4 + warp;
  if (y >= 2 * c.kv_heads) return;
  const bool is_v = y >= c.kv_heads;
  const int head = is_v ? y - c.kv_heads : y;
  const bool rot = !is_v && p.cos_table != nullptr;
  const int64_t slots = static_cast<int64_t>(c.num_blocks) * bs;
  const int sub = lane / kLanes;

  for (int i = 0; i < tokens; ++i) {
    const int slot = slot_of[1 + i];
    if (slot < 0 || slot >= slots) continue;
    const int block = slot / bs, off = slot % bs;
    if (off > 0 && slot_of[i] == slot - 1) continue;  // inside a run
    // the run ends with the block or where a slot does not follow
    int len = bs - off;
    for (int b = 1; b < len; b += 32) {
      const bool stop = b + lane < len && slot_of[1 + i + b + lane] != slot + b + lane;
      const uint32_t m = __ballot_sync(~0u, stop);
      if (m) {
        len = b + __ffs(m) - 1;
        break;
      }
    }
    const int64_t t = t0 + i;
    const T* x0 = qkv + t * p.ld_qkv + static_cast<int64_t>(p.q_heads + y) * D + chunk * 8;
    float* scale_at = (is_v ? c.v_scale : c.k_scale) + static_cast<int64_t>(block) * c.kv_heads + head;
    const float old = off > 0 ? *scale_at : 0.f;

    auto turn = [&](int j, float* lo, float* hi) {
      if (!rot) return;
      const int pos = pos_of[1 + i + j];
      float cs[8], sn[8];
      load_f8(p.cos_table + static_cast<int64_t>(pos) * half + chunk * 8, cs);
      load_f8(p.sin_table + static_cast<int64_t>(pos) * half + chunk * 8, sn);
      rotate8(lo, hi, cs, sn);
    };
    // |x| as bits: ordered like the values, with infinity and NaN on top
    uint32_t top = 0;
    uint4 w[kPasses][2];
    auto fetch = [&](int j0) {
#pragma unroll
      for (int e = 0; e < kPasses; ++e) {
        const int j = j0 + e * kTokens + sub;
        if (j < len) {
          w[e][0] = *reinterpret_cast<const uint4*>(x0 + j * p.ld_qkv);
          w[e][1] = *reinterpret_cast<const uint4*>(x0 + j * p.ld_qkv + half);
        }
      }
    };
    for (int j0 = 0; j0 < len; j0 += kTokens * kPasses) {
      fetch(j0);
#pragma unroll
      for (int e = 0; e < kPasses; ++e) {
        const int j = j0 + e * kTokens + sub;
        if (j < len) {
          float lo[8], hi[8];
          unpack8(w[e][0], lo, T());
          unpack8(w[e][1], hi, T());
          turn(j, lo, hi);
#pragma unroll
          for (int b = 0; b < 8; ++b)
            top = max(top, max(__float_as_uint(lo[b]) & 0x7fffffffu, __float_as_uint(hi[b]) & 0x7fffffffu));
        }
      }
    }
    top = __reduce_max_sync(~0u, top);
    const float fresh = top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), 127.f) : __uint_as_float(0x7fc00000u);
    const float s = isnan(old) || isnan(fresh) ? __uint_as_float(0x7fc00000u) : fmaxf(old, fresh);
    if (lane == 0) *scale_at = s;

    int8_t* base = (is_v ? c.v : c.k) + (static_cast<int64_t>(block) * c.kv_heads + head) * bs * D;
    if (off > 0 && s > old && old > 0.f) {
      const float ratio = __fdiv_rn(old, s);
      uint4* levels = reinterpret_cast<uint4*>(base);
#pragma unroll 4
      for (int k = lane; k < off * D / 16; k += 32) {
        uint4 w = levels[k];
        uint32_t* e = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t m[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) m[b] = level_bits(level_of(e[j], b) * ratio);
          e[j] = pack_bytes(m);
        }
        levels[k] = w;
      }
    }
    const float inv = s > 1.2e-38f && s < 8e37f ? __frcp_rn(s) : 0.f;
    for (int j0 = 0; j0 < len; j0 += kTokens * kPasses) {
      fetch(j0);
#pragma unroll
      for (int e = 0; e < kPasses; ++e) {
        const int j = j0 + e * kTokens + sub;
        if (j < len) {
          uint2 wl = make_uint2(0, 0), wh = make_uint2(0, 0);
          if (s > 0.f) {
            float lo[8], hi[8];
            unpack8(w[e][0], lo, T());
            unpack8(w[e][1], hi, T());
            turn(j, lo, hi);
            wl = make_uint2(pack_levels(lo, s, inv), pack_levels(lo + 4, s, inv));
            wh = make_uint2(pack_levels(hi, s, inv), pack_levels(hi + 4, s, inv));
          }
          int8_t* o = base + (off + j) * D + chunk * 8;
          *reinterpret_cast<uint2*>(o) = wl;
          *reinterpret_cast<uint2*>(o + half) = wh;
        }
      }
    }
    i += len - 1;
  }
}

// A CTA per block and head, of keys (y = 0) or values; a thread per 16 levels.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Kv8ReadParams p) {
  const Kv8Cache& c = p.cache;
  const int n = c.block_size * c.dim / 16;
  const bool is_v = blockIdx.y != 0;
  const uint32_t heads = c.kv_heads, i = blockIdx.x / heads, head = blockIdx.x - i * heads;
  grid_dep_wait();
  grid_dep_launch();
  const int id = p.blocks[i];
  const bool there = id >= 0 && id < c.num_blocks;
  const int64_t row = there ? static_cast<int64_t>(id) * c.kv_heads + head : 0;
  const float s = there ? (is_v ? c.v_scale : c.k_scale)[row] : 0.f;
  const uint4* src = reinterpret_cast<const uint4*>(is_v ? c.v : c.k) + row * n;
  T* dst = static_cast<T*>(is_v ? p.v_out : p.k_out) + static_cast<int64_t>(blockIdx.x) * n * 16;
#pragma unroll 4
  for (int k = threadIdx.x; k < n; k += kThreads) {
    const uint4 w = there ? src[k] : make_uint4(0, 0, 0, 0);
    const uint32_t e[4] = {w.x, w.y, w.z, w.w};
    float f[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = level_of(e[j >> 2], j & 3) * s;
    store8(dst + k * 16, f);
    store8(dst + k * 16 + 8, f + 8);
  }
}

bool misaligned(const void* p, uintptr_t by) { return (reinterpret_cast<uintptr_t>(p) & (by - 1)) != 0; }

}  // namespace

const char* kv8_cache_problem(const Kv8Cache& c) {
  if (c.num_blocks < 0 || c.kv_heads <= 0) return "cache sizes must be positive";
  if (c.dim != 64 && c.dim != 128) return "head size must be 64 or 128";
  if (c.block_size != 16 && c.block_size != 32 && c.block_size != 64 && c.block_size != 128)
    return "block size must be 16, 32, 64 or 128";
  if (static_cast<int64_t>(c.num_blocks) * c.block_size > INT32_MAX ||
      static_cast<int64_t>(c.num_blocks) * c.kv_heads > INT32_MAX)
    return "slots are 32-bit: too many blocks";
  if (c.num_blocks > 0 && (!c.k || !c.v || !c.k_scale || !c.v_scale)) return "null operand";
  if (misaligned(c.k, 16) || misaligned(c.v, 16)) return "levels must be 16-byte aligned";
  return nullptr;
}

cudaError_t kv8_append_launch(const Kv8AppendParams& p, cudaStream_t stream, const char** err) {
  *err = kv8_cache_problem(p.cache);
  const int64_t heads = static_cast<int64_t>(p.q_heads) + 2 * static_cast<int64_t>(p.cache.kv_heads);
  if (!*err && (p.tokens < 0 || p.tokens > INT32_MAX || p.q_heads < 0)) *err = "sizes out of range";
  if (!*err && p.type != kKvF16 && p.type != kKvBF16) *err = "element type must be f16 or bf16";
  if (*err) return cudaErrorInvalidValue;
  if (p.tokens == 0) return cudaSuccess;
  const bool rot = p.cos_table != nullptr;
  if (!p.qkv || !p.slots || (rot && (!p.sin_table || !p.positions || (p.q_heads > 0 && !p.q_out))))
    *err = "null operand";
  else if (p.ld_qkv < heads * p.cache.dim || p.ld_qkv % 8 != 0 || misaligned(p.qkv, 16))
    *err = "qkv rows must hold all heads, 16-byte aligned";
  else if (rot && (p.table_rows <= 0 || misaligned(p.cos_table, 16) || misaligned(p.sin_table, 16) ||
                   misaligned(p.q_out, 16)))
    *err = "cos, sin and q_out must be 16-byte aligned and not empty";
  if (*err) return cudaErrorInvalidValue;
  // decode steps spread over the GPU token by token; prompts take a block's worth of tokens, mostly one run, at a time
  const int seg = p.tokens >= 2048 ? p.cache.block_size : p.tokens >= 512 ? 4 : 1;
  const int64_t kv_blocks = (p.tokens + seg - 1) / seg * ((2 * static_cast<int64_t>(p.cache.kv_heads) + 3) / 4);
  const int64_t per_block = kThreads / (p.cache.dim / 16) * kQPasses;
  const int64_t q_blocks = rot ? (p.tokens * p.q_heads + per_block - 1) / per_block : 0;
  if (kv_blocks + q_blocks > INT32_MAX || p.tokens * p.q_heads > INT32_MAX) *err = "too many tokens and heads";
  if (*err) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(kv_blocks + q_blocks));
  auto kern = p.cache.dim == 128 ? (p.type == kKvF16 ? append_kernel<__half, 128> : append_kernel<__nv_bfloat16, 128>)
                                 : (p.type == kKvF16 ? append_kernel<__half, 64> : append_kernel<__nv_bfloat16, 64>);
  return launch_dependent(kern, grid, dim3(kThreads), 0, stream, p, seg, static_cast<int>(kv_blocks));
}

cudaError_t kv8_read_launch(const Kv8ReadParams& p, cudaStream_t stream, const char** err) {
  *err = kv8_cache_problem(p.cache);
  if (!*err && p.count < 0) *err = "negative size";
  if (!*err && p.type != kKvF16 && p.type != kKvBF16) *err = "element type must be f16 or bf16";
  if (*err) return cudaErrorInvalidValue;
  if (p.count == 0) return cudaSuccess;
  if (!p.blocks || !p.k_out || !p.v_out) *err = "null operand";
  else if (misaligned(p.k_out, 16) || misaligned(p.v_out, 16)) *err = "outputs must be 16-byte aligned";
  if (*err) return cudaErrorInvalidValue;
  const int64_t pairs = static_cast<int64_t>(p.count) * p.cache.kv_heads;
  if (pairs > INT32_MAX) {
    *err = "too many blocks";
    return cudaErrorInvalidValue;
  }
  return launch_dependent(p.type == kKvF16 ? read_kernel<__half> : read_kernel<__nv_bfloat16>,
                          dim3(static_cast<unsigned>(pairs), 2), dim3(kThreads), 0, stream, p);
}

}  // namespace disc_b200
