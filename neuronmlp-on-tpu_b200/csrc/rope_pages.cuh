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

// Pairs of 16-bit elements in one word.
template <typename T>
SVD_DEV uint32_t pack_pair(float lo, float hi);
template <>
SVD_DEV uint32_t pack_pair<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
SVD_DEV uint32_t pack_pair<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <typename T>
SVD_DEV float2 unpack_pair(uint32_t v);
template <>
SVD_DEV float2 unpack_pair<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
SVD_DEV float2 unpack_pair<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

// ------------------------------------------------------------------- rotary
struct RopeParams {
  int tokens, q_heads, kv_heads, head_dim, half;
  int block_size;
  int tile;                              // tokens per CTA, at most kRopeTile
  int rot_units, head_units, v_units;    // pieces: turned, all of a head of q or k; of a head of v
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
// Tokens per CTA, and tokens whose loads a thread has in flight (measured at
// 8192 tokens of 32 and 8 heads of 128, us: tiles of 4, 8, 16 38.8, 40.6, 44.1;
// batches of 2, 4, 8 in tiles of 8 39.5, 40.6, 41.7).
constexpr int kRopeTile = 4;
constexpr int kRopeBatch = 4;

// E elements of 2 bytes: one 16-byte vector, or one element.
template <int E>
struct alignas(E * 2) RopeVec {
  uint32_t w[E / 2];
};
template <>
struct alignas(2) RopeVec<1> {
  uint16_t w[1];
};

// (a cos - b sin, b cos + a sin) for E pairs; turn[e * stride] holds pair e's
// cosine and sine.  Pairs are (a[e], b[e]), or neighbours in a then b.
template <typename T, int E, bool INTER>
SVD_DEV void rope_turn(RopeVec<E>& a, RopeVec<E>& b, const float2* turn, int stride) {
  if constexpr (E == 1) {
    T x = *reinterpret_cast<T*>(&a.w[0]), y = *reinterpret_cast<T*>(&b.w[0]);
    const float2 r = turn[0];
    const float fx = elem_to_float(x), fy = elem_to_float(y);
    x = elem_from_float<T>(fx * r.x - fy * r.y);
    y = elem_from_float<T>(fy * r.x + fx * r.y);
    a.w[0] = *reinterpret_cast<uint16_t*>(&x);
    b.w[0] = *reinterpret_cast<uint16_t*>(&y);
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      if constexpr (INTER) {
        const float2 u = unpack_pair<T>(a.w[i]), v = unpack_pair<T>(b.w[i]);
        const float2 r = turn[i * stride], t = turn[(E / 2 + i) * stride];
        a.w[i] = pack_pair<T>(u.x * r.x - u.y * r.y, u.y * r.x + u.x * r.y);
        b.w[i] = pack_pair<T>(v.x * t.x - v.y * t.y, v.y * t.x + v.x * t.y);
      } else {
        const float2 u = unpack_pair<T>(a.w[i]), v = unpack_pair<T>(b.w[i]);
        const float2 r = turn[2 * i * stride], t = turn[(2 * i + 1) * stride];
        a.w[i] = pack_pair<T>(u.x * r.x - v.x * r.y, u.y * t.x - v.y * t.y);
        b.w[i] = pack_pair<T>(v.x * r.x + u.x * r.y, v.y * t.x + u.y * t.y);
      }
    }
  }
}

// Rotary positions and the cache write, fp32, rounded once.  A CTA takes a tile
// of tokens.  A thread takes the same piece of a head (E elements copied, or 2 E
// turned) for every token of the tile, so that its place is worked out once, and
// has the loads of kRopeBatch tokens in flight; the cosines and sines, computed
// once for all heads, come between the first loads and their use.  The angle in
// turns, position * inv_freq / 2 pi, is reduced in fp64, so a position of 10^6
// loses nothing.  Memory-bound: q, k, v are read once and every output written
// once, 218 MB in 38.8 us = 5.6 TB/s at 8192 tokens of 32 and 8 heads of 128;
// with a piece's place worked out for each token anew the instructions bound it
// (half of the issue slots, 59 us).
template <typename T, int E, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  using Vec = RopeVec<E>;
  extern __shared__ float2 turns[];  // [tile][pair % E][pair / E]
  __shared__ long long k_at[kRopeTile], v_at[kRopeTile];  // where each token goes in the caches, or -1
  grid_dependency_wait();  // no early launch of the next kernel: its waiting CTAs would take this one's places
  const int t0 = blockIdx.x * p.tile;
  const int nt = min(p.tile, p.tokens - t0);
  const int qk_units = (p.q_heads + p.kv_heads) * p.head_units;
  const int units = qk_units + (p.k_cache != nullptr ? p.kv_heads * p.v_units : 0);
  bool begun = false;
  for (int w = threadIdx.x; w < units || !begun; w += kRopeThreads) {
    // the piece: where it lies in the source, the output and the cache
    const T* src = nullptr;
    T *dst = nullptr, *put = nullptr;
    long long src_step = 0, dst_step = 0;
    const long long* at = k_at;
    int second = 0;     // from a to b, in elements; 0: copied
    int unit = 0;
    if (w < qk_units) {
      int h = w / p.head_units;
      unit = w - h * p.head_units;
      int lo;
      if (unit < p.rot_units) {
        lo = INTER ? 2 * unit * E : unit * E;
        second = INTER ? E : p.half;
      } else {
        lo = 2 * p.half + (unit - p.rot_units) * E;
      }
      if (h < p.q_heads) {
        src = static_cast<const T*>(p.q) + t0 * p.q_token + h * p.q_head + lo;
        src_step = p.q_token;
        dst_step = static_cast<long long>(p.q_heads) * p.head_dim;
        dst = static_cast<T*>(p.q_out) + t0 * dst_step + h * p.head_dim + lo;
      } else {
        h -= p.q_heads;
        src = static_cast<const T*>(p.k) + t0 * p.k_token + h * p.k_head + lo;
        src_step = p.k_token;
        if (p.k_out != nullptr) {
          dst_step = static_cast<long long>(p.kv_heads) * p.head_dim;
          dst = static_cast<T*>(p.k_out) + t0 * dst_step + h * p.head_dim + lo;
        }
        if (p.k_cache != nullptr) put = static_cast<T*>(p.k_cache) + static_cast<long long>(h) * p.block_size * p.head_dim + lo;
      }
    } else if (w < units) {
      const int x = w - qk_units, h = x / p.v_units, lo = (x - h * p.v_units) * E;
      src = static_cast<const T*>(p.v) + t0 * p.v_token + h * p.v_head + lo;
      src_step = p.v_token;
      put = static_cast<T*>(p.v_cache) + static_cast<long long>(h) * p.block_size * p.head_dim + lo;
      at = v_at;
    }
    for (int b0 = 0; b0 < nt; b0 += kRopeBatch) {
      Vec a[kRopeBatch], b[kRopeBatch];
#pragma unroll
      for (int i = 0; i < kRopeBatch; ++i) {
        if (src != nullptr && b0 + i < nt) {
          a[i] = *reinterpret_cast<const Vec*>(src + (b0 + i) * src_step);
          if (second != 0) b[i] = *reinterpret_cast<const Vec*>(src + (b0 + i) * src_step + second);
        }
      }
      if (!begun) {  // every thread once, whatever pieces it has
        begun = true;
        for (int i = threadIdx.x; i < nt * p.half; i += kRopeThreads) {
          const int t = i / p.half, j = i - t * p.half;
          const double angle = static_cast<double>(p.positions[t0 + t]) * static_cast<double>(p.inv_freq[j]) *
                               0.15915494309189533577;  // in turns: 1 / (2 pi)
          float s, c;
          sincospif(static_cast<float>(2.0 * (angle - rint(angle))), &s, &c);
          turns[t * p.half + (j % E) * p.rot_units + j / E] = make_float2(c * p.scale, s * p.scale);
        }
        if (static_cast<int>(threadIdx.x) < nt) {
          long long slot = p.k_cache != nullptr ? p.slots[t0 + threadIdx.x] : -1;
          if (slot >= p.cache_slots) slot = -1;
          const long long block = slot >= 0 ? slot / p.block_size : 0, place = slot - block * p.block_size;
          k_at[threadIdx.x] = slot >= 0 ? block * p.k_block + place * p.head_dim : -1;
          v_at[threadIdx.x] = slot >= 0 ? block * p.v_block + place * p.head_dim : -1;
        }
        __syncthreads();
      }
      if (src == nullptr) break;
#pragma unroll
      for (int i = 0; i < kRopeBatch; ++i) {
        const int t = b0 + i;
        if (t < nt) {
          if (second != 0) rope_turn<T, E, INTER>(a[i], b[i], turns + t * p.half + unit, p.rot_units);
          if (dst != nullptr) {
            *reinterpret_cast<Vec*>(dst + t * dst_step) = a[i];
            if (second != 0) *reinterpret_cast<Vec*>(dst + t * dst_step + second) = b[i];
          }
          if (put != nullptr && at[t] >= 0) {
            *reinterpret_cast<Vec*>(put + at[t]) = a[i];
            if (second != 0) *reinterpret_cast<Vec*>(put + at[t] + second) = b[i];
          }
        }
      }
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
// itself, so no CTA waits for another's table entries.  Lengths are not trusted:
// a request ends at 2^31 - 1 tokens, and the sums stop there, so that no place
// is ever worked out of a wrapped one; a chunk with a length of kPagesCalm or more is
// added up one by one.  Latency-bound: one scan and one bisection stand between
// the loads and the stores; 2.5 us for 8 requests of one token, 4.1 us for 1024
// with up to 300 each (in a CUDA graph).

constexpr int kPagesCalm = 1 << 21;  // lengths and widths below it have sums below 2^31 over a chunk

// a + b for a, b >= 0, at most 2^31 - 1.
SVD_DEV int capped_sum(int a, int b) { return static_cast<int>(min(static_cast<unsigned>(a) + static_cast<unsigned>(b), 0x7fffffffu)); }

// Tokens held and added of one request, and the blocks that it has and lacks.
struct PagesRequest {
  int held, added, have, lacks;
};
SVD_DEV PagesRequest load_request(const PagesParams& p, int b) {
  PagesRequest r{0, 0, 0, 0};
  if (b < p.batch) {
    r.held = max(p.held[b], 0);
    r.added = min(max(p.added[b], 0), 0x7fffffff - r.held);
  }
  const unsigned size = p.block_size, up = size - 1;
  r.have = static_cast<int>(min((r.held + up) / size, static_cast<unsigned>(p.width)));
  r.lacks = static_cast<int>(min((r.held + r.added + up) / size, static_cast<unsigned>(p.width))) - r.have;
  return r;
}

__global__ void __launch_bounds__(kPagesThreads) page_step_kernel(const PagesParams p) {
  constexpr int PER = kPagesChunk / kPagesThreads;
  __shared__ int s_cu[kPagesChunk + 1];    // first new token of each request of the chunk
  __shared__ int s_take[kPagesChunk + 1];  // blocks taken before it
  __shared__ int s_held[kPagesChunk];
  __shared__ unsigned long long s_warp[kPagesThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int left = max(0, min(*p.free_count, p.capacity));
  int cu0 = 0, take0 = 0;  // carried over the chunks
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // places among the tokens and blocks of a chunk; unsigned, as a stride may go beyond 2^31
  const unsigned first = blockIdx.x * kPagesThreads + threadIdx.x, stride = gridDim.x * kPagesThreads;
  const auto table_page = [&](int b, int have, int take, int idx) -> int {
    if (idx >= p.width) return -1;
    if (idx < have) return p.table[b * p.ld_table + idx];
    const int at = capped_sum(take, idx - have);
    return at < left ? p.free_blocks[left - 1 - at] : -1;
  };
  for (int b0 = 0; b0 < p.batch; b0 += kPagesChunk) {
    // running sums, (blocks << 32 | tokens) in one word; each thread owns PER requests in a row
    unsigned long long mine[PER], sum = 0;
    int held[PER];
    bool wild = p.width >= kPagesCalm;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const PagesRequest r = load_request(p, b0 + threadIdx.x * PER + i);
      wild = wild || r.added >= kPagesCalm;
      held[i] = r.held;
      mine[i] = sum;
      sum += static_cast<unsigned long long>(r.lacks) << 32 | static_cast<unsigned>(r.added);
    }
    unsigned long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) s_warp[warp] = inc;
    int cu1 = 0, take1 = 0;
    const bool calm = __syncthreads_or(wild) == 0;
    if (calm) {
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
        s_cu[threadIdx.x * PER + i] = capped_sum(cu0, static_cast<int>(at & 0xffffffffu));
        s_take[threadIdx.x * PER + i] = capped_sum(take0, static_cast<int>(at >> 32));
        s_held[threadIdx.x * PER + i] = held[i];
      }
      cu1 = capped_sum(cu0, static_cast<int>(all & 0xffffffffu));
      take1 = capped_sum(take0, static_cast<int>(all >> 32));
      if (threadIdx.x == 0) s_cu[kPagesChunk] = cu1;
    } else if (threadIdx.x == 0) {  // sums that the halves of a word may not hold: one after another
      int cu = cu0, take = take0;
      for (int i = 0; i < kPagesChunk; ++i) {
        const PagesRequest r = load_request(p, b0 + i);
        s_cu[i] = cu;
        s_take[i] = take;
        s_held[i] = r.held;
        cu = capped_sum(cu, r.added);
        take = capped_sum(take, r.lacks);
      }
      s_cu[kPagesChunk] = cu;
      s_take[kPagesChunk] = take;
    }
    __syncthreads();

    const int here = min(kPagesChunk, p.batch - b0);
    if (!calm) {
      cu1 = s_cu[kPagesChunk];
      take1 = s_take[kPagesChunk];
    }
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; i < here; i += kPagesThreads) {
        p.cu[b0 + i] = s_cu[i];
        p.lens[b0 + i] = s_held[i] + (s_cu[i + 1] - s_cu[i]);
      }
    }
    // the last request of the chunk that begins at or before x
    const auto request_of = [&](const int* begins, int x) -> int {
      int lo = 0, hi = here;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (begins[mid] <= x) lo = mid;
        else hi = mid;
      }
      return lo;
    };
    const auto have_of = [&](int lo) -> int {
      const unsigned size = p.block_size;
      return static_cast<int>(min((s_held[lo] + (size - 1)) / size, static_cast<unsigned>(p.width)));
    };
    const unsigned end = cu1 > p.tokens ? p.tokens : cu1;
    for (unsigned t = cu0 + first; t < end; t += stride) {
      const int lo = request_of(s_cu, static_cast<int>(t));
      const int pos = s_held[lo] + (static_cast<int>(t) - s_cu[lo]);
      const int idx = pos / p.block_size, off = pos - idx * p.block_size;
      const int have = have_of(lo), page = table_page(b0 + lo, have, s_take[lo], idx);
      if (t < static_cast<unsigned>(p.tokens)) {  // always; without the question the loads come later (2.71 for 2.53 us)
        p.slots[t] = page >= 0 ? static_cast<long long>(page) * p.block_size + off : -1;
        p.positions[t] = pos;
      }
      // the first token of a new block enters it into the table
      if (idx >= have && idx < p.width && off == 0) p.table[(b0 + lo) * p.ld_table + idx] = page;
    }
    if (cu1 > p.tokens) {  // more tokens than the caller said: their blocks by themselves
      for (unsigned x = take0 + first; x < static_cast<unsigned>(take1); x += stride) {
        const int lo = request_of(s_take, static_cast<int>(x));
        const int have = have_of(lo), idx = have + (static_cast<int>(x) - s_take[lo]);
        if (idx < p.width) p.table[(b0 + lo) * p.ld_table + idx] = table_page(b0 + lo, have, s_take[lo], idx);
      }
    }
    cu0 = cu1;
    take0 = take1;
    __syncthreads();
  }
  for (unsigned t = cu0 + first; t < static_cast<unsigned>(p.tokens); t += stride) {
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
