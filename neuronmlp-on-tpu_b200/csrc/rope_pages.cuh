// Rotary positions with the cache write, and the paging step: the two kernels
// around attention that only move data.
#pragma once

#include "ptx.cuh"

namespace svdmlp {

template <typename T>
SVD_DEV float elem_to_float(T v);
template <>
SVD_DEV float elem_to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
SVD_DEV float elem_to_float<__half>(__half v) { return __half2float(v); }
template <typename T>
SVD_DEV T elem_from_float(float v);
template <>
SVD_DEV __nv_bfloat16 elem_from_float<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <>
SVD_DEV __half elem_from_float<__half>(float v) { return __float2half(v); }

// ------------------------------------------------------------------- rotary
struct RopeParams {
  int tokens, q_heads, kv_heads, head_dim, half, interleaved;
  int block_size, block_shift;  // shift: log2(block_size), or -1 when it is no power of two
  int tile;                     // tokens per CTA
  float scale;
  const void *q, *k, *v;
  long long q_token, q_head, k_token, k_head, v_token, v_head;
  const int* positions;
  const long long* slots;
  const float* inv_freq;
  void *q_out, *k_out, *k_cache, *v_cache;
  long long k_block, v_block, cache_slots;
};

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxTile = 16;

template <typename T, int E>
struct alignas(E * 2) ElemVec {
  T x[E];
};

// out = (a cos - b sin, b cos + a sin) per pair, fp32, rounded once.  A CTA
// takes a tile of tokens: their cosines and sines are computed once into
// shared memory (the angle in turns, position * inv_freq / 2 pi, is reduced in
// fp64, so a position of 10^6 loses nothing), then every head of q, k and v is
// cut into units of E (copied) or 2E (turned) elements that the threads walk
// through; E = 8 moves 16-byte vectors, E = 1 serves any alignment.
// Memory-bound: q, k, v are read once and every output written once.
template <typename T, int E>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  extern __shared__ float2 turn[];  // [tile][half]
  using Vec = ElemVec<T, E>;
  grid_dependency_wait();  // no early launch of the next kernel: its waiting CTAs would take this one's places
  const int t0 = blockIdx.x * p.tile;
  const int nt = min(p.tile, p.tokens - t0);
  for (int i = threadIdx.x; i < nt * p.half; i += kRopeThreads) {
    const int t = i / p.half, j = i - t * p.half;
    const double turns = static_cast<double>(p.positions[t0 + t]) * static_cast<double>(p.inv_freq[j]) *
                         0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    turn[i] = make_float2(c * p.scale, s * p.scale);
  }
  __syncthreads();

  const bool cached = p.k_cache != nullptr;
  const int rot_units = p.half / E;                                   // per head, 2E elements each
  const int head_units = rot_units + (p.head_dim - 2 * p.half) / E;   // of a head of q or k
  const int v_units = cached ? p.head_dim / E : 0;
  const int qk_units = (p.q_heads + p.kv_heads) * head_units;
  const int token_units = qk_units + p.kv_heads * v_units;
  for (int u = threadIdx.x; u < nt * token_units; u += kRopeThreads) {
    const int t = u / token_units;
    int w = u - t * token_units;
    const long long token = t0 + t;
    long long slot = -1;
    long long place = 0, block = 0;
    if (cached) {
      slot = p.slots[token];
      if (slot >= p.cache_slots) slot = -1;
      if (slot >= 0) {
        block = p.block_shift >= 0 ? slot >> p.block_shift : slot / p.block_size;
        place = slot - block * p.block_size;
      }
    }
    if (w >= qk_units) {  // a piece of v
      w -= qk_units;
      const int h = w / v_units, d = (w - h * v_units) * E;
      if (slot >= 0) {
        const Vec x = *reinterpret_cast<const Vec*>(static_cast<const T*>(p.v) + token * p.v_token + h * p.v_head + d);
        *reinterpret_cast<Vec*>(static_cast<T*>(p.v_cache) + block * p.v_block +
                                (h * static_cast<long long>(p.block_size) + place) * p.head_dim + d) = x;
      }
      continue;
    }
    const int qk_head = w / head_units;
    const int unit = w - qk_head * head_units;
    const bool is_q = qk_head < p.q_heads;
    const int h = is_q ? qk_head : qk_head - p.q_heads;
    const T* src = is_q ? static_cast<const T*>(p.q) + token * p.q_token + h * p.q_head
                        : static_cast<const T*>(p.k) + token * p.k_token + h * p.k_head;
    T* dst = is_q ? static_cast<T*>(p.q_out) + (token * p.q_heads + h) * p.head_dim
                  : p.k_out != nullptr ? static_cast<T*>(p.k_out) + (token * p.kv_heads + h) * p.head_dim : nullptr;
    T* put = !is_q && slot >= 0 ? static_cast<T*>(p.k_cache) + block * p.k_block +
                                      (h * static_cast<long long>(p.block_size) + place) * p.head_dim
                                : nullptr;
    if (unit < rot_units) {
      const int lo = p.interleaved ? 2 * unit * E : unit * E;
      const int hi = p.interleaved ? lo + E : lo + p.half;
      Vec a = *reinterpret_cast<const Vec*>(src + lo), b = *reinterpret_cast<const Vec*>(src + hi);
      float x[2 * E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[e] = elem_to_float(a.x[e]);
        x[E + e] = elem_to_float(b.x[e]);
      }
      const float2* cs = turn + t * p.half + unit * E;
      if (p.interleaved) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 r = cs[e];
          const float even = x[2 * e], odd = x[2 * e + 1];
          x[2 * e] = even * r.x - odd * r.y;
          x[2 * e + 1] = odd * r.x + even * r.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 r = cs[e];
          const float first = x[e], second = x[E + e];
          x[e] = first * r.x - second * r.y;
          x[E + e] = second * r.x + first * r.y;
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        a.x[e] = elem_from_float<T>(x[e]);
        b.x[e] = elem_from_float<T>(x[E + e]);
      }
      if (dst != nullptr) {
        *reinterpret_cast<Vec*>(dst + lo) = a;
        *reinterpret_cast<Vec*>(dst + hi) = b;
      }
      if (put != nullptr) {
        *reinterpret_cast<Vec*>(put + lo) = a;
        *reinterpret_cast<Vec*>(put + hi) = b;
      }
    } else {
      const int d = 2 * p.half + (unit - rot_units) * E;
      const Vec x = *reinterpret_cast<const Vec*>(src + d);
      if (dst != nullptr) *reinterpret_cast<Vec*>(dst + d) = x;
      if (put != nullptr) *reinterpret_cast<Vec*>(put + d) = x;
    }
  }
}

// ------------------------------------------------------------------- paging
struct PagesParams {
  int batch, tokens, block_size, width, capacity;
  int* table;
  long long ld_table;
  const int *held, *added, *free_blocks, *free_count;
  long long* slots;
  int *positions, *cu, *lens, *count_out, *missing;
};

constexpr int kPagesThreads = 256;
constexpr int kPagesChunk = 1024;  // requests scanned at a time

// Every CTA scans the requests, kPagesChunk at a time: running sums of the
// tokens they add and of the blocks they lack, in shared memory.  The new
// tokens of the chunk are then spread over all threads of the grid, each one
// finding its request by bisection; CTA 0 writes what there is one of per
// request.  A token in a new block takes the block's number from the free list
// itself, so no CTA waits for another's table entries.  Latency-bound: one
// scan and one bisection stand between the loads and the stores.
__global__ void __launch_bounds__(kPagesThreads) page_step_kernel(const PagesParams p) {
  constexpr int PER = kPagesChunk / kPagesThreads;
  __shared__ int s_cu[kPagesChunk + 1];    // first new token of each request of the chunk
  __shared__ int s_take[kPagesChunk];      // blocks taken before it
  __shared__ int s_held[kPagesChunk];
  __shared__ unsigned long long s_warp[kPagesThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int left = max(0, min(*p.free_count, p.capacity));
  int cu0 = 0, take0 = 0;  // carried over the chunks
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const auto table_page = [&](int b, int have, int take, int idx) -> int {
    if (idx >= p.width) return -1;
    if (idx < have) return p.table[b * p.ld_table + idx];
    const int at = take + idx - have;
    return at < left ? p.free_blocks[left - 1 - at] : -1;
  };
  for (int b0 = 0; b0 < p.batch; b0 += kPagesChunk) {
    // running sums, (blocks << 32 | tokens) in one word; each thread owns PER requests in a row
    unsigned long long mine[PER], sum = 0;
    int held[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = b0 + threadIdx.x * PER + i;
      int h = 0, n = 0;
      if (b < p.batch) {
        h = max(p.held[b], 0);
        n = max(p.added[b], 0);
      }
      held[i] = h;
      const int have = min((h + p.block_size - 1) / p.block_size, p.width);
      const int need = min((h + n + p.block_size - 1) / p.block_size, p.width);
      mine[i] = sum;
      sum += static_cast<unsigned long long>(need - have) << 32 | static_cast<unsigned>(n);
    }
    unsigned long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    unsigned long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPagesThreads / 32; ++w) {
      if (w < warp) before += s_warp[w];
      all += s_warp[w];
    }
    before += inc - sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned long long at = before + mine[i];
      s_cu[threadIdx.x * PER + i] = cu0 + static_cast<int>(at & 0xffffffffu);
      s_take[threadIdx.x * PER + i] = take0 + static_cast<int>(at >> 32);
      s_held[threadIdx.x * PER + i] = held[i];
    }
    const int cu1 = cu0 + static_cast<int>(all & 0xffffffffu), take1 = take0 + static_cast<int>(all >> 32);
    if (threadIdx.x == 0) s_cu[kPagesChunk] = cu1;
    __syncthreads();

    const int here = min(kPagesChunk, p.batch - b0);
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; i < here; i += kPagesThreads) {
        p.cu[b0 + i] = s_cu[i];
        p.lens[b0 + i] = s_held[i] + s_cu[i + 1] - s_cu[i];
      }
    }
    for (int t = cu0 + blockIdx.x * kPagesThreads + threadIdx.x; t < cu1; t += gridDim.x * kPagesThreads) {
      int lo = 0, hi = here;  // the last request that starts at or before t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t) lo = mid;
        else hi = mid;
      }
      const int pos = s_held[lo] + t - s_cu[lo];
      const int idx = pos / p.block_size, off = pos - idx * p.block_size;
      const int have = min((s_held[lo] + p.block_size - 1) / p.block_size, p.width);
      const int page = table_page(b0 + lo, have, s_take[lo], idx);
      if (t < p.tokens) {
        p.slots[t] = page >= 0 ? static_cast<long long>(page) * p.block_size + off : -1;
        p.positions[t] = pos;
      }
      // the first token of a new block enters it into the table
      if (idx >= have && idx < p.width && off == 0) p.table[(b0 + lo) * p.ld_table + idx] = page;
    }
    cu0 = cu1;
    take0 = take1;
    __syncthreads();
  }
  for (int t = cu0 + blockIdx.x * kPagesThreads + threadIdx.x; t < p.tokens; t += gridDim.x * kPagesThreads) {
    p.slots[t] = -1;
    p.positions[t] = 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.cu[p.batch] = cu0;
    *p.count_out = max(left - take0, 0);
    *p.missing = max(take0 - left, 0);
  }
}

}  // namespace svdmlp
