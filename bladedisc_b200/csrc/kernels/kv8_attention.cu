// Attention over the 8-bit paged cache:
//   s_ij = scale * k_scale[block(j)] * (q_i . k_j),   j <= kv_len - q_len + i
//   o_i  = sum_j softmax(s_i)_j * v_scale[block(j)] * v_j,   0 where row i sees no key.
#include "kv8.h"

#include "device_info.h"
#include "kv8_types.cuh"
#include "sm100_ptx.cuh"

namespace disc_b200 {

__device__ int g_kv8_status = 0;

namespace {

constexpr int kThreads = 128;

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// One CTA per token, query head and request: a thread per key of a group of 128 for the scores, a thread per
// output column for the values.
template <typename T>
__global__ void __launch_bounds__(kThreads) plain_kernel(Kv8AttentionParams p) {
  const Kv8Cache& c = p.cache;
  const int D = c.dim, bs = c.block_size;
  const int r = blockIdx.z, h = blockIdx.y, i = blockIdx.x;
  __shared__ float q[128], w[kThreads], red[8];
  grid_dep_wait();
  grid_dep_launch();
  const int q_len = p.q_lens[r];
  const int64_t row = static_cast<int64_t>(p.q_start[r]) + i;
  if (i >= q_len || row < 0 || row >= p.tokens) return;
  const int kv_len = min(max(p.kv_lens[r], 0), p.table_width * bs);
  const int64_t keys = min(static_cast<int64_t>(kv_len), static_cast<int64_t>(kv_len) - q_len + i + 1);
  const int head = h / (p.q_heads / c.kv_heads);
  if (threadIdx.x < D)
    q[threadIdx.x] = to_float(static_cast<const T*>(p.q)[row * p.ld_q + h * D + threadIdx.x]) * p.scale;
  __syncthreads();
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int64_t k0 = 0; k0 < keys; k0 += kThreads) {
    const int64_t j = k0 + threadIdx.x;
    float s = -INFINITY, vs = 0.f;
    int id = -1;
    if (j < keys) id = p.table[static_cast<int64_t>(r) * p.table_width + j / bs];
    const bool there = id >= 0 && id < c.num_blocks;
    if (there) {
      const int64_t bh = static_cast<int64_t>(id) * c.kv_heads + head;
      const int8_t* k = c.k + (bh * bs + j % bs) * D;
      float a = 0.f;
      for (int d = 0; d < D; ++d) a += q[d] * static_cast<float>(k[d]);
      s = a * c.k_scale[bh];
      vs = c.v_scale[bh];
    }
    float top = s;
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mn = fmaxf(m, top);
    const float e = there ? expf(s - (mn == -INFINITY ? 0.f : mn)) : 0.f;
    float sum = e;
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
    if ((threadIdx.x & 31) == 0) red[4 + (threadIdx.x >> 5)] = sum;
    w[threadIdx.x] = there ? e * vs : 0.f;
    __syncthreads();
    const float keep = m == -INFINITY ? 0.f : expf(m - mn);
    l = l * keep + (red[4] + red[5] + red[6] + red[7]);
    m = mn;
    if (threadIdx.x < D) {
      o *= keep;
      for (int64_t x = 0; x < kThreads && k0 + x < keys; ++x) {
        const int b = p.table[static_cast<int64_t>(r) * p.table_width + (k0 + x) / bs];
        if (b < 0 || b >= c.num_blocks) continue;
        o += w[x] * static_cast<float>(
                        c.v[((static_cast<int64_t>(b) * c.kv_heads + head) * bs + (k0 + x) % bs) * D + threadIdx.x]);
      }
    }
    __syncthreads();
  }
  if (threadIdx.x < D) {
    T* out = static_cast<T*>(p.out) + row * p.ld_out + h * D + threadIdx.x;
    *out = static_cast<T>(l == 0.f ? 0.f : o / l);
  }
}

bool misaligned(const void* p, uintptr_t by) { return (reinterpret_cast<uintptr_t>(p) & (by - 1)) != 0; }

template <typename T>
cudaError_t launch_t(const Kv8AttentionParams& p, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.max_q), static_cast<unsigned>(p.q_heads),
                  static_cast<unsigned>(p.requests));
  return launch_dependent(plain_kernel<T>, grid, dim3(kThreads), 0, stream, p);
}

}  // namespace

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
  return p.type == kKvF16 ? launch_t<__half>(p, stream) : launch_t<__nv_bfloat16>(p, stream);
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
