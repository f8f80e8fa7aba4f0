// Block tables and slot maps of the paged cache, built on the device from request lengths, so that a decode
// loop that is replayed from a CUDA graph never asks the host where a token goes.
//
// extend: every request asks for n new tokens; blocks come off the top of a stack of free blocks in the order
// (request, place); a request whose blocks are not there, whose table row is full or whose tokens fall behind
// the slot array gets nothing (slot -1, lengths unchanged).  trim gives the blocks behind the kept tokens back
// in the reverse order, so that trim(old lengths) undoes an extend bit for bit.
//
// The work is two prefix sums over at most 8192 requests and one pass over tokens, so latency is what counts:
// one launch, one cluster.  Every CTA of the cluster computes all the sums (a few hundred ns; cheaper than
// handing them over), a cluster barrier separates the last read of the state from its first update, and the
// tokens are dealt over all threads.
#include "kv8.h"

#include "device_info.h"
#include "sm100_ptx.cuh"

namespace disc_b200 {
namespace {

constexpr int kThreads = 1024;
constexpr int kItems = kKvMaxRequests / kThreads;

struct Sums {
  int64_t warp[32];
};

// Inclusive prefix sum over the block of one value per thread.
__device__ __forceinline__ int64_t block_inclusive(int64_t v, Sums& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) s.warp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int64_t w = s.warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(~0u, w, o);
      if (lane >= o) w += u;
    }
    s.warp[lane] = w;
  }
  __syncthreads();
  if (warp > 0) v += s.warp[warp - 1];
  __syncthreads();  // the sums may be overwritten by the next call
  return v;
}

// Last index i of [0, n) with start[i] <= t; start[0] <= t.
__device__ __forceinline__ int last_not_above(const int32_t* start, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int clamp_len(int v, int64_t room) {
  return v < 0 ? 0 : (v > room ? static_cast<int>(room) : v);
}

__global__ void __launch_bounds__(kThreads, 1) extend_kernel(KvBlocksParams p) {
  extern __shared__ int32_t dyn[];
  __shared__ Sums sums;
  const int R = p.requests, bs = p.block_size;
  int32_t* start = dyn;          // [R + 1] first token row of a request
  int32_t* first = start + R + 1;  // [R] blocks handed out before this request
  int32_t* had = first + R;      // [R] cached tokens before, or -1 - that when the request is not served
  const int items = (R + kThreads - 1) / kThreads;
  const int64_t room = static_cast<int64_t>(p.table_width) * bs;
  grid_dep_wait();
  grid_dep_launch();

  const int count = min(max(*p.free_count, 0), p.num_blocks);
  int n[kItems], len[kItems];
  int64_t total = 0;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int r = threadIdx.x * items + i;
    n[i] = len[i] = 0;
    if (i < items && r < R) {
      n[i] = max(p.tokens[r], 0);
      len[i] = clamp_len(p.lens[r], room);
    }
    total += n[i];
  }
  const int64_t end0 = block_inclusive(total, sums);
  int64_t at = end0 - total;
  int64_t needs = 0;
  int need[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int r = threadIdx.x * items + i;
    need[i] = -1;  // no room
    if (i < items && r < R) {
      start[r] = static_cast<int32_t>(at < INT32_MAX ? at : INT32_MAX);
      at += n[i];
      if (static_cast<int64_t>(len[i]) + n[i] <= room && at <= p.max_tokens)
        need[i] = static_cast<int>((static_cast<int64_t>(len[i]) + n[i] + bs - 1) / bs - (len[i] + bs - 1) / bs);
      needs += max(need[i], 0);
      if (r == R - 1) start[R] = static_cast<int32_t>(at < INT32_MAX ? at : INT32_MAX);
    }
  }
  int64_t upto = block_inclusive(needs, sums) - needs;
  int64_t given_here = 0;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int r = threadIdx.x * items + i;
    if (i < items && r < R) {
      // (what was asked for before a refused request can only have been refused for the same reason or not
      // at all, so that `first` is right for every request that is served)
      first[r] = static_cast<int32_t>(upto < INT32_MAX ? upto : INT32_MAX);
      upto += max(need[i], 0);
      const bool served = need[i] == 0 || (need[i] > 0 && upto <= count);
      had[r] = served ? len[i] : -1 - len[i];
      if (!served) n[i] = 0;
      given_here += served ? need[i] : 0;
    }
  }
  const int64_t given = block_inclusive(given_here, sums);  // ends with a barrier: the arrays are complete
  cluster_sync_all();  // every CTA has read the state: it may change now

  const uint32_t rank = cluster_ctarank();
  if (rank == 0) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int r = threadIdx.x * items + i;
      if (i < items && r < R) {
        const int kv = len[i] + n[i];
        p.lens[r] = kv;
        p.kv_lens[r] = kv;
        p.q_lens[r] = n[i];
        p.q_start[r] = start[r];
      }
    }
    if (threadIdx.x == kThreads - 1) {
      p.q_start[R] = start[R];
      *p.free_count = static_cast<int32_t>(count - given);
    }
  }

  const int asked = start[R];
  for (int64_t t = rank * kThreads + threadIdx.x; t < p.max_tokens; t += gridDim.x * kThreads) {
    int slot = -1, pos = -1;
    if (t < asked) {
      const int r = last_not_above(start, R, static_cast<int>(t));
      if (had[r] >= 0) {
        pos = had[r] + static_cast<int>(t) - start[r];
        const int b = pos / bs, held = (had[r] + bs - 1) / bs;
        int32_t* entry = p.table + static_cast<int64_t>(r) * p.table_width + b;
        int id;
        if (b >= held) {
          id = p.free_list[count - 1 - (first[r] + b - held)];
          if (pos % bs == 0) *entry = id;  // the first token of a block enters it into the table
        } else {
          id = *entry;
        }
        slot = id >= 0 && id < p.num_blocks ? id * bs + pos % bs : -1;
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

__global__ void __launch_bounds__(kThreads, 1) trim_kernel(KvBlocksParams p) {
  extern __shared__ int32_t dyn[];
  __shared__ Sums sums;
  const int R = p.requests, bs = p.block_size;
  int32_t* base = dyn;       // [R + 1] blocks freed before this request
  int32_t* stay = base + R + 1;  // [R] blocks that the request keeps
  const int items = (R + kThreads - 1) / kThreads;
  const int64_t room = static_cast<int64_t>(p.table_width) * bs;
  grid_dep_wait();
  grid_dep_launch();

  const int count = min(max(*p.free_count, 0), p.num_blocks);
  int keep[kItems], freed[kItems];
  int64_t total = 0;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int r = threadIdx.x * items + i;
    keep[i] = freed[i] = 0;
    if (i < items && r < R) {
      const int len = clamp_len(p.lens[r], room);
      keep[i] = min(max(p.tokens[r], 0), len);
      stay[r] = (keep[i] + bs - 1) / bs;
      freed[i] = (len + bs - 1) / bs - stay[r];
    }
    total += freed[i];
  }
  const int64_t end0 = block_inclusive(total, sums);
  int64_t at = end0 - total;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int r = threadIdx.x * items + i;
    if (i < items && r < R) {
      base[r] = static_cast<int32_t>(at);
      at += freed[i];
      if (r == R - 1) base[R] = static_cast<int32_t>(at);
    }
  }
  __syncthreads();
  cluster_sync_all();

  const uint32_t rank = cluster_ctarank();
  const int gone = base[R];
  if (rank == 0) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int r = threadIdx.x * items + i;
      if (i < items && r < R) p.lens[r] = keep[i];
    }
    if (threadIdx.x == 0) *p.free_count = min(count + gone, p.num_blocks);
  }
  for (int f = rank * kThreads + threadIdx.x; f < gone; f += gridDim.x * kThreads) {
    const int r = last_not_above(base, R, f);
    int32_t* entry = p.table + static_cast<int64_t>(r) * p.table_width + stay[r] + (f - base[r]);
    const int place = count + gone - 1 - f;
    if (place < p.num_blocks) p.free_list[place] = *entry;
    *entry = -1;
  }
}

const char* problem(const KvBlocksParams& p) {
  if (p.requests < 0 || p.requests > kKvMaxRequests) return "requests must be 0 .. 8192";
  if (p.block_size <= 0 || p.table_width < 0 || p.num_blocks < 0) return "negative size";
  if (static_cast<int64_t>(p.num_blocks) * p.block_size > INT32_MAX ||
      static_cast<int64_t>(p.table_width) * p.block_size > INT32_MAX ||
      static_cast<int64_t>(p.table_width) * p.requests > INT32_MAX)
    return "slots are 32-bit: num_blocks * block_size, table_width * block_size and requests * table_width must fit";
  if (p.requests > 0 && (!p.tokens || !p.lens)) return "null operand";
  if (p.requests > 0 && p.table_width > 0 && !p.table) return "null operand";
  if (!p.free_count || (p.num_blocks > 0 && !p.free_list)) return "null operand";
  return nullptr;
}

cudaError_t launch(void (*kern)(KvBlocksParams), const KvBlocksParams& p, int ctas, size_t smem, cudaStream_t stream) {
  if (smem > 48 * 1024) {
    const cudaError_t st =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (st != cudaSuccess) return st;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

// One CTA while its threads have one item each; the portable cluster of eight beyond that.
int ctas_for(int64_t items) { return items <= kThreads ? 1 : 8; }

}  // namespace

cudaError_t kv_blocks_extend_launch(const KvBlocksParams& p, cudaStream_t stream, const char** err) {
  *err = problem(p);
  if (!*err && p.max_tokens < 0) *err = "negative size";
  if (!*err && (!p.q_start || (p.requests > 0 && (!p.q_lens || !p.kv_lens)) ||
                (p.max_tokens > 0 && (!p.slots || !p.positions))))
    *err = "null operand";
  if (*err) return cudaErrorInvalidValue;
  if (p.requests == 0) {
    cudaError_t st = cudaMemsetAsync(p.q_start, 0, sizeof(int32_t), stream);
    if (st == cudaSuccess && p.max_tokens > 0) {
      st = cudaMemsetAsync(p.slots, 0xff, sizeof(int32_t) * static_cast<size_t>(p.max_tokens), stream);
      if (st == cudaSuccess)
        st = cudaMemsetAsync(p.positions, 0xff, sizeof(int32_t) * static_cast<size_t>(p.max_tokens), stream);
    }
    return st;
  }
  return launch(extend_kernel, p, ctas_for(p.max_tokens), sizeof(int32_t) * (3 * static_cast<size_t>(p.requests) + 1),
                stream);
}

cudaError_t kv_blocks_trim_launch(const KvBlocksParams& p, cudaStream_t stream, const char** err) {
  *err = problem(p);
  if (*err) return cudaErrorInvalidValue;
  if (p.requests == 0) return cudaSuccess;
  return launch(trim_kernel, p, ctas_for(static_cast<int64_t>(p.requests) * p.table_width),
                sizeof(int32_t) * (2 * static_cast<size_t>(p.requests) + 1), stream);
}

}  // namespace disc_b200
