// Attention one row at a time: a warp per (query row, head) walks the keys it
// sees with a running maximum and sum.  The simplest form that is right for
// every case; every key and value is read once per row, so it is bound by L2.
#pragma once

#include "rope_pages.cuh"

namespace svdmlp {

// One warp's running softmax over keys, each lane holding head_dim / 32
// elements of the query and of the output.
template <int E>
struct RowState {
  float q[E], o[E], m, l;
};

template <typename T, int E>
SVD_DEV void row_init(RowState<E>& r, const T* q, float scale) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    r.q[e] = elem_to_float(q[lane_id() * E + e]) * scale;
    r.o[e] = 0.f;
  }
  r.m = -INFINITY;
  r.l = 0.f;
}

template <typename T, int E>
SVD_DEV void row_key(RowState<E>& r, const T* k, const T* v) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) s += r.q[e] * elem_to_float(k[lane_id() * E + e]);
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const float m = fmaxf(r.m, s);
  const float base = m == -INFINITY ? 0.f : m;
  const float c = __expf(r.m - base), w = __expf(s - base);
  r.m = m;
  r.l = r.l * c + w;
#pragma unroll
  for (int e = 0; e < E; ++e) r.o[e] = r.o[e] * c + w * elem_to_float(v[lane_id() * E + e]);
}

template <typename T, int E>
SVD_DEV void row_store(const RowState<E>& r, T* out) {
  const float inv = r.l > 0.f ? 1.f / r.l : (r.l == 0.f ? 0.f : r.l);
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane_id() * E + e] = elem_from_float<T>(r.l == 0.f ? 0.f : r.o[e] * inv);
}

// The request that holds row t: the last b with cu[b] <= t, when t < cu[b + 1].
SVD_DEV int find_request(const int* cu, int batch, int t) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return t >= cu[lo] && t < cu[lo + 1] ? lo : -1;
}

template <typename T, int D>
__global__ void prompt_rows_kernel(const svdmlp_prompt_args p) {
  constexpr int E = D / 32;
  const long long w = (blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x) >> 5;
  if (w >= static_cast<long long>(p.q_tokens) * p.q_heads) return;
  const int t = static_cast<int>(w / p.q_heads), h = static_cast<int>(w % p.q_heads);
  const int b = find_request(p.cu_q, p.batch, t);
  RowState<E> r;
  row_init<T>(r, static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head, p.scale);
  if (b >= 0) {
    const int k0 = max(p.cu_k[b], 0), k1 = min(p.cu_k[b + 1], p.k_tokens);
    const int last = p.causal ? min(k1, p.cu_k[b + 1] - (p.cu_q[b + 1] - t) + 1) : k1;
    const int hk = h / (p.q_heads / p.kv_heads);
    for (int j = k0; j < last; ++j)
      row_key<T>(r, static_cast<const T*>(p.k) + j * p.k_token + hk * p.k_head,
                 static_cast<const T*>(p.v) + j * p.v_token + hk * p.v_head);
  }
  row_store<T>(r, static_cast<T*>(p.out) + t * p.out_token + h * p.out_head);
}

template <typename T, int D>
__global__ void tree_rows_kernel(const svdmlp_tree_args p) {
  constexpr int E = D / 32;
  const long long w = (blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x) >> 5;
  if (w >= static_cast<long long>(p.tokens) * p.q_heads) return;
  const int t = static_cast<int>(w / p.q_heads), h = static_cast<int>(w % p.q_heads);
  const int b = find_request(p.cu_q, p.batch, t);
  RowState<E> r;
  row_init<T>(r, static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head, p.scale);
  if (b >= 0) {
    const int row = t - p.cu_q[b], n = p.cu_q[b + 1] - p.cu_q[b];
    const int len = min(static_cast<long long>(p.lens[b]), static_cast<long long>(p.table_width) * p.block_size);
    const int first = p.lens[b] - n;  // the tree's first key
    const int hk = h / (p.q_heads / p.kv_heads);
    const unsigned long long mask = p.mask != nullptr ? p.mask[t] : 0;
    for (int j = 0; j < len; ++j) {
      const int node = j - first;
      if (node >= 0 && (p.mask != nullptr ? node >= 64 || !(mask >> node & 1) : node > row)) continue;
      const int page = p.table[b * p.ld_table + j / p.block_size];
      if (page < 0 || page >= p.num_blocks) continue;
      const long long at = (hk * static_cast<long long>(p.block_size) + j % p.block_size) * D;
      row_key<T>(r, static_cast<const T*>(p.k_cache) + page * p.k_block + at,
                 static_cast<const T*>(p.v_cache) + page * p.v_block + at);
    }
  }
  row_store<T>(r, static_cast<T*>(p.out) + t * p.out_token + h * p.out_head);
}

}  // namespace svdmlp
