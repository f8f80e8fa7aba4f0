// Block tables and slot maps of the paged cache, built on the device from request lengths, so that a decode
// loop that is replayed from a CUDA graph never asks the host where a token goes.
//
// extend: every request asks for n new tokens; blocks come off the top of a stack of free blocks in the order
// (request, place); a request whose blocks are not there, whose table row is full or whose tokens fall behind
// the slot array gets nothing (slot -1, lengths unchanged).  trim gives the blocks behind the kept tokens back
// in the reverse order, so that trim(old lengths) undoes an extend bit for bit.
//
// The work is two prefix sums over at most 8192 requests and one pass over tokens, so latency is what counts:
// one launch, one cluster, as few threads as the batch needs (barriers cost with every warp).  Every CTA of the
// cluster computes all the sums (a few hundred ns; cheaper than handing them over), a cluster barrier separates the
// last read of the state from its first update, and the tokens are dealt over all threads.  Prompts have more tokens
// than one cluster writes quickly (112600: 24 us): there it only makes the table, and a second kernel over the whole
// GPU writes the slots (10 us in all).  Extending 64 requests by one token each and trimming them
// again takes 7.8 us on the GPU, all of it latency: the launch and the chain lengths, sums, table, slot.
#include "kv8.h"

#include <algorithm>

#include "device_info.h"
#include "sm100_ptx.cuh"

namespace disc_b200 {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kItems = kKvMaxRequests / kMaxThreads;  // requests per thread at most

struct Sums {
  int64_t warp[32];
};

// Inclusive prefix sum over the block of one value per thread.
__device__ __forceinline__ int64_t block_inclusive(int64_t v, Sums& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) s.warp[warp] = v;
  __syncthreads();
  if (warps <= 8) {
    for (int w = 0; w < warp; ++w) v += s.warp[w];
  } else {
    if (warp == 0) {
      int64_t w = lane < warps ? s.warp[lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(~0u, w, o);
        if (lane >= o) w += u;
      }
      s.warp[lane] = w;
    }
    __syncthreads();
    if (warp > 0) v += s.warp[warp - 1];
  }
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

// tokens <= 2^31 - 1 and a block of at most as many: no overflow in unsigned arithmetic
__device__ __forceinline__ int blocks_of(int tokens, int bs) {
  return static_cast<int>((static_cast<uint32_t>(tokens) + static_cast<uint32_t>(bs) - 1) / static_cast<uint32_t>(bs));
}

__device__ __forceinline__ int clamp_len(int v, int64_t room) {
  return v < 0 ? 0 : (v > room ? static_cast<int>(room) : v);
}

template <bool SLOTS>
__global__ void __launch_bounds__(kMaxThreads, 1) extend_kernel(KvBlocksParams p) {
  extern __shared__ int32_t dyn[];
  __shared__ Sums sums, sums2;
  __shared__ int given;
  const int R = p.requests, bs = p.block_size;
  const int threads = blockDim.x;
  int32_t* start = dyn;          // [R + 1] first token row of a request
  int32_t* first = start + R + 1;  // [R] blocks handed out before this request
  int32_t* had = first + R;      // [R] cached tokens before, or -1 - that when the request is not served
  const int items = (R + threads - 1) / threads;
  const int64_t room = static_cast<int64_t>(p.table_width) * bs;
  grid_dep_wait();
  grid_dep_launch();

  const int count = min(max(*p.free_count, 0), p.num_blocks);
  if (threadIdx.x == 0) given = 0;
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
        need[i] = blocks_of(len[i] + n[i], bs) - blocks_of(len[i], bs);
      needs += max(need[i], 0);
      if (r == R - 1) start[R] = static_cast<int32_t>(at < INT32_MAX ? at : INT32_MAX);
    }
  }
  int64_t upto = block_inclusive(needs, sums2) - needs;
  int last = 0;  // blocks handed out up to the last served request of this thread
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
      if (served && need[i] > 0) last = static_cast<int>(upto);
    }
  }
  last = __reduce_max_sync(~0u, last);
  if ((threadIdx.x & 31) == 0 && last > 0) atomicMax(&given, last);
  __syncthreads();  // the arrays are complete
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
    if (threadIdx.x == threads - 1) {
      p.q_start[R] = start[R];
      *p.free_count = count - given;
    }
  }

  if (!SLOTS) {
    for (int f = rank * threads + threadIdx.x; f < given; f += gridDim.x * threads) {
      const int r = last_not_above(first, R, f);  // of requests with the same sum the last one takes blocks
      p.table[static_cast<int64_t>(r) * p.table_width + blocks_of(had[r], bs) + f - first[r]] =
          p.free_list[count - 1 - f];
    }
    return;
  }
  const int asked = start[R];
  for (int t = rank * threads + threadIdx.x; t < p.max_tokens; t += gridDim.x * threads) {
    int slot = -1, pos = -1;
    if (t < asked) {
      const int r = last_not_above(start, R, t);
      if (had[r] >= 0) {
        pos = had[r] + t - start[r];
        const int b = pos / bs, held = blocks_of(had[r], bs);
        int32_t* entry = p.table + static_cast<int64_t>(r) * p.table_width + b;
        int id;
        if (b >= held) {
          id = p.free_list[count - 1 - (first[r] + b - held)];
          if (pos - b * bs == 0) *entry = id;  // the first token of a block enters it into the table
        } else {
          id = *entry;
        }
        slot = id >= 0 && id < p.num_blocks ? id * bs + pos - b * bs : -1;
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

// Slots and positions from what extend_kernel wrote, four consecutive tokens per thread.
constexpr int kSlotThreads = 256;
__global__ void __launch_bounds__(kSlotThreads) slots_kernel(KvBlocksParams p) {
  const int R = p.requests, bs = p.block_size;
  grid_dep_wait();
  grid_dep_launch();
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kSlotThreads + threadIdx.x) * 4;
  if (t0 >= p.max_tokens) return;
  const int asked = p.q_start[R];
  int pos[4], id[4], off[4], slot[4];
  int r = t0 < asked ? last_not_above(p.q_start, R, static_cast<int>(t0)) : R;
  int end = r < R ? p.q_start[r + 1] : 0, n = r < R ? p.q_lens[r] : 0;
  int q = r < R ? p.kv_lens[r] - n + static_cast<int>(t0) - p.q_start[r] : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + i;
    pos[i] = -1;
    off[i] = 0;
    id[i] = -1;
    if (t < asked) {
      if (t >= end) {  // the next request that has tokens
        while (t >= end) end = p.q_start[++r + 1];
        n = p.q_lens[r];
        q = p.kv_lens[r] - n;
      }
      if (n > 0) {
        pos[i] = q;
        const int b = q / bs;
        off[i] = q - b * bs;
        id[i] = p.table[static_cast<int64_t>(r) * p.table_width + b];
      }
      ++q;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) slot[i] = id[i] >= 0 && id[i] < p.num_blocks ? id[i] * bs + off[i] : -1;
  if (t0 + 4 <= p.max_tokens && ((reinterpret_cast<uintptr_t>(p.slots) | reinterpret_cast<uintptr_t>(p.positions)) & 15) == 0) {
    *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t0 + i < p.max_tokens) {
        p.slots[t0 + i] = slot[i];
        p.positions[t0 + i] = pos[i];
      }
    }
  }
}

__global__ void __launch_bounds__(kMaxThreads, 1) trim_kernel(KvBlocksParams p) {
  extern __shared__ int32_t dyn[];
  __shared__ Sums sums;
  const int R = p.requests, bs = p.block_size;
  const int threads = blockDim.x;
  int32_t* base = dyn;       // [R + 1] blocks freed before this request
  int32_t* stay = base + R + 1;  // [R] blocks that the request keeps
  const int items = (R + threads - 1) / threads;
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
      stay[r] = blocks_of(keep[i], bs);
      freed[i] = blocks_of(len, bs) - stay[r];
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
  for (int f = rank * threads + threadIdx.x; f < gone; f += gridDim.x * threads) {
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

// Shared memory of a kernel with `arrays` values per request, and one.
size_t smem_of(int arrays, int requests) { return sizeof(int32_t) * (arrays * static_cast<size_t>(requests) + 1); }

template <void (*kern)(KvBlocksParams), int ARRAYS>
cudaError_t launch(const KvBlocksParams& p, int ctas, int threads, cudaStream_t stream) {
  const size_t smem = smem_of(ARRAYS, p.requests);
  if (smem > 48 * 1024) {
    static std::atomic<uint64_t> ready{0};
    const cudaError_t st = allow_smem(kern, static_cast<int>(smem_of(ARRAYS, kKvMaxRequests)), ready);
    if (st != cudaSuccess) return st;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
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

// Threads of a CTA for this many requests or tokens; requests beyond go several to a thread.
int threads_for(int64_t n) { return n <= 256 ? 256 : n <= 512 ? 512 : kMaxThreads; }

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
  if (p.max_tokens <= 8 * kMaxThreads) {  // a token per thread
    return launch<extend_kernel<true>, 3>(p, p.max_tokens <= kMaxThreads ? 1 : 8,
                                          threads_for(std::max(p.requests, p.max_tokens)), stream);
  }
  const cudaError_t st =
      launch<extend_kernel<false>, 3>(p, 8, threads_for(std::max(p.requests, p.num_blocks / 8)), stream);
  if (st != cudaSuccess) return st;
  const int64_t blocks = (static_cast<int64_t>(p.max_tokens) + 4 * kSlotThreads - 1) / (4 * kSlotThreads);
  return launch_dependent(slots_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kSlotThreads), 0, stream, p);
}

cudaError_t kv_blocks_trim_launch(const KvBlocksParams& p, cudaStream_t stream, const char** err) {
  *err = problem(p);
  if (*err) return cudaErrorInvalidValue;
  if (p.requests == 0) return cudaSuccess;
  const int64_t most = static_cast<int64_t>(p.requests) * p.table_width;  // blocks that can come back
  return launch<trim_kernel, 2>(p, most <= 8 * kMaxThreads ? 1 : 8,
                                threads_for(std::max<int64_t>(p.requests, most / 4)), stream);
}

}  // namespace disc_b200
