// Append to the 8-bit cache and reading blocks back.
//
// A block of tokens and a head share one scale s = max|x| / 127 over the tokens stored so far, levels are
// rne(x / s).  When new tokens raise the maximum of a block that already holds tokens, those are moved to the
// new scale: level' = rne(level * (s_old / s)); the error that adds is at most half a level each time the maximum
// grows.  Keys are rotated (pairs (i, i + dim / 2)) in fp32 and quantized without a rounding in between.
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

__device__ __forceinline__ uint32_t pack_levels(const float* x, float s) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float l = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -127.f), 127.f);
    w |= (static_cast<uint32_t>(static_cast<int>(l)) & 0xffu) << (8 * i);
  }
  return w;
}

// Grid: x = segments of `seg` consecutive tokens; y = kv_heads keys, kv_heads values, then groups of four query
// heads.  A run is a maximal sequence of consecutive tokens whose slots are consecutive inside one block; the
// CTA whose segment holds its first token works on all of it, once for the maximum and once for the levels (the
// second read comes from the caches).
template <typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(Kv8AppendParams p, int seg) {
  const Kv8Cache& c = p.cache;
  const int D = c.dim, bs = c.block_size, half = D / 2;
  const int chunks = D / 16;               // threads per token: eight values of each half of the head
  const int per_pass = kThreads / chunks;  // tokens per pass of the CTA
  const int chunk = threadIdx.x % chunks, sub = threadIdx.x / chunks;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * seg;
  const int64_t t1 = min(t0 + seg, p.tokens);
  const T* qkv = static_cast<const T*>(p.qkv);
  grid_dep_wait();
  grid_dep_launch();

  const int y = blockIdx.y;
  if (y >= 2 * c.kv_heads) {
    const int h0 = (y - 2 * c.kv_heads) * 4, h1 = min(h0 + 4, p.q_heads);
    T* out = static_cast<T*>(p.q_out);
    for (int64_t t = t0 + sub; t < t1; t += per_pass) {
      const int pos = min(max(p.positions[t], 0), p.table_rows - 1);
      float cs[8], sn[8], lo[8], hi[8];
      load_f8(p.cos_table + static_cast<int64_t>(pos) * half + chunk * 8, cs);
      load_f8(p.sin_table + static_cast<int64_t>(pos) * half + chunk * 8, sn);
      for (int h = h0; h < h1; ++h) {
        const T* x = qkv + t * p.ld_qkv + h * D + chunk * 8;
        load8(x, lo);
        load8(x + half, hi);
        rotate8(lo, hi, cs, sn);
        T* o = out + (t * p.q_heads + h) * D + chunk * 8;
        store8(o, lo);
        store8(o + half, hi);
      }
    }
    return;
  }

  const bool is_v = y >= c.kv_heads;
  const int head = is_v ? y - c.kv_heads : y;
  const bool rot = !is_v && p.cos_table != nullptr;
  const T* x0 = qkv + static_cast<int64_t>(p.q_heads + y) * D + chunk * 8;
  const int64_t slots = static_cast<int64_t>(c.num_blocks) * bs;
  __shared__ uint32_t red[kThreads / 32];

  for (int64_t t = t0; t < t1; ++t) {
    const int64_t slot = p.slots[t];
    if (slot < 0 || slot >= slots) continue;
    const int block = static_cast<int>(slot / bs), off = static_cast<int>(slot % bs);
    if (t > 0 && off > 0 && p.slots[t - 1] == slot - 1) continue;  // inside a run
    int len = 1;
    while (off + len < bs && t + len < p.tokens && p.slots[t + len] == slot + len) ++len;

    auto load = [&](int i, float* lo, float* hi) {
      const T* x = x0 + (t + i) * p.ld_qkv;
      load8(x, lo);
      load8(x + half, hi);
      if (rot) {
        const int pos = min(max(p.positions[t + i], 0), p.table_rows - 1);
        float cs[8], sn[8];
        load_f8(p.cos_table + static_cast<int64_t>(pos) * half + chunk * 8, cs);
        load_f8(p.sin_table + static_cast<int64_t>(pos) * half + chunk * 8, sn);
        rotate8(lo, hi, cs, sn);
      }
    };
    // |x| as bits: ordered like the values, with infinity and NaN on top
    uint32_t top = 0;
    for (int i = sub; i < len; i += per_pass) {
      float lo[8], hi[8];
      load(i, lo, hi);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = max(top, __float_as_uint(lo[e]) & 0x7fffffffu);
        top = max(top, __float_as_uint(hi[e]) & 0x7fffffffu);
      }
    }
    top = __reduce_max_sync(~0u, top);
    __syncthreads();  // `red` of the run before has been read
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    float* scale_at = (is_v ? c.v_scale : c.k_scale) + static_cast<int64_t>(block) * c.kv_heads + head;
    const float old = off > 0 ? *scale_at : 0.f;
    __syncthreads();
    top = max(max(red[0], red[1]), max(red[2], red[3]));
    const float fresh = top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), 127.f) : __uint_as_float(0x7fc00000u);
    const float s = isnan(old) || isnan(fresh) ? __uint_as_float(0x7fc00000u) : fmaxf(old, fresh);
    if (threadIdx.x == 0) *scale_at = s;

    int8_t* base = (is_v ? c.v : c.k) + (static_cast<int64_t>(block) * c.kv_heads + head) * bs * D;
    if (off > 0 && s > old && old > 0.f) {
      const float ratio = __fdiv_rn(old, s);
      uint4* levels = reinterpret_cast<uint4*>(base);
      for (int i = threadIdx.x; i < off * D / 16; i += kThreads) {
        uint4 w = levels[i];
        uint32_t* e = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t m = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            m |= (static_cast<uint32_t>(__float2int_rn(level_of(e[j], b) * ratio)) & 0xffu) << (8 * b);
          e[j] = m;
        }
        levels[i] = w;
      }
    }
    for (int i = sub; i < len; i += per_pass) {
      uint2 wl = make_uint2(0, 0), wh = make_uint2(0, 0);
      if (s > 0.f) {
        float lo[8], hi[8];
        load(i, lo, hi);
        wl = make_uint2(pack_levels(lo, s), pack_levels(lo + 4, s));
        wh = make_uint2(pack_levels(hi, s), pack_levels(hi + 4, s));
      }
      int8_t* o = base + (off + i) * D + chunk * 8;
      *reinterpret_cast<uint2*>(o) = wl;
      *reinterpret_cast<uint2*>(o + half) = wh;
    }
    t += len - 1;
  }
}

// One thread per 16 levels.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(Kv8ReadParams p) {
  const Kv8Cache& c = p.cache;
  const int64_t per_head = static_cast<int64_t>(c.block_size) * c.dim;
  const int64_t n = static_cast<int64_t>(p.count) * c.kv_heads * per_head / 16;
  grid_dep_wait();
  grid_dep_launch();
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < 2 * n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const bool is_v = i >= n;
    const int64_t at = (is_v ? i - n : i) * 16;
    const int64_t bh = at / per_head;
    const int64_t id = p.blocks[bh / c.kv_heads], head = bh % c.kv_heads;
    float f[16];
    if (id >= 0 && id < c.num_blocks) {
      const int64_t row = id * c.kv_heads + head;
      const float s = (is_v ? c.v_scale : c.k_scale)[row];
      const uint4 w = *reinterpret_cast<const uint4*>((is_v ? c.v : c.k) + row * per_head + at % per_head);
      const uint32_t* e = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
      for (int j = 0; j < 16; ++j) f[j] = level_of(e[j >> 2], j & 3) * s;
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) f[j] = 0.f;
    }
    T* o = static_cast<T*>(is_v ? p.v_out : p.k_out) + at;
    store8(o, f);
    store8(o + 8, f + 8);
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
  const int64_t gy = 2 * static_cast<int64_t>(p.cache.kv_heads) + (rot ? (p.q_heads + 3) / 4 : 0);
  if (!*err && gy > 65535) *err = "too many heads";
  if (*err) return cudaErrorInvalidValue;
  const int seg = p.tokens >= 2048 ? 16 : p.tokens >= 512 ? 4 : 1;
  const dim3 grid(static_cast<unsigned>((p.tokens + seg - 1) / seg), static_cast<unsigned>(gy));
  return p.type == kKvF16 ? launch_dependent(append_kernel<__half>, grid, dim3(kThreads), 0, stream, p, seg)
                          : launch_dependent(append_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, stream, p, seg);
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
  const int64_t items = 2 * static_cast<int64_t>(p.count) * p.cache.kv_heads * p.cache.block_size * p.cache.dim / 16;
  int64_t grid = (items + kThreads - 1) / kThreads;
  const int64_t cap = static_cast<int64_t>(device_sm_count()) * 16;
  if (grid > cap) grid = cap;
  return p.type == kKvF16
             ? launch_dependent(read_kernel<__half>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, p)
             : launch_dependent(read_kernel<__nv_bfloat16>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0,
                                stream, p);
}

}  // namespace disc_b200
