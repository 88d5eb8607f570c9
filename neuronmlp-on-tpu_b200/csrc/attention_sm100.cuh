// Attention on tcgen05, for packed prompts and for the newest tokens over a
// paged cache:  out = softmax(scale q k^T) v  per query head, the softmax in
// one pass over the keys with a running maximum and sum.
//
// Rows.  A query tile is 128 rows of one key/value head: all gp query heads of
// the group for tt = 128 / gp tokens, row = token * gp + head (a group of more
// than 64 heads is taken head by head).  Packing the group lets one tile of k
// and v serve every head that shares it, fills the 128 rows of the MMA when
// there are few tokens, and narrows the causal diagonal to tt tokens.
//
// A unit is one (request, head group, token tile) of two row tiles ("pair"), or
// of one row tile whose key steps alternate between the two softmax groups
// ("alt", for requests of at most 128 rows, where a second row tile would be
// empty).  Its keys are walked in steps of 128.
//
// Work.  All steps of all units form one line, cut into equal pieces, one per
// CTA (persistent, one per SM): every CTA computes the cut itself from the
// request lengths on the device, so ragged lengths, long prompts and a single
// long context load every SM alike.  A unit that a cut divides leaves fp32
// partials (maximum, sum, unnormalised output) in the workspace; the CTA that
// arrives last at the unit's counter joins them in the order of the keys, so
// results do not depend on the order of arrival.
//
// Roles (384 threads): two softmax warpgroups, one thread per row; an MMA warp;
// a TMA warp.  TMEM (512 columns): scores S0, S1 (128 each; the probabilities
// overwrite them as 16-bit pairs and are the A operand of the second product)
// and outputs O0, O1.  The MMA warp issues P0 V(j), Q0 K(j+1), P1 V(j),
// Q1 K(j+1): while one group turns scores into probabilities, the tensor pipe
// works for the other.  The output is rescaled only when a row's maximum grows
// by more than 8 (in powers of two): a stale base keeps probabilities below
// 2^8, which the 16-bit types and the fp32 sums hold without loss.
//
// What bounds it: at 128 keys x 128 rows a step costs 1024 cycles of the
// tensor pipe (head_dim 128) and 1024 of the exponential unit; with few rows
// the bytes of k and v.
#pragma once

#include <type_traits>

#include "rope_pages.cuh"

namespace svdmlp {

constexpr int kAttnThreads = 384;
constexpr int kAttnStep = 128;        // keys per step
constexpr int kAttnMaxGrid = 512;     // counters and partial slots reserved
constexpr float kAttnLazy = 8.0f;     // growth of the maximum (log2) that a stale base absorbs

struct AttnParams {
  int batch, q_tokens, k_tokens;
  int head_groups, gp, group;         // units per token tile; query heads per unit; query heads per kv head
  int tt, alt, causal, tree;
  int min_steps;                      // fewest steps a CTA takes
  float c;                            // |scale| log2(e)
  int neg;                            // scale < 0
  const int *cu_q, *cu_k;             // packed keys
  const int *lens, *table;            // paged keys
  const long long* mask;
  long long ld_table;
  int block_size, block_shift, num_blocks, width;
  const void *q, *k, *v;              // for the row-wise path
  long long q_token, q_head, k_token, k_head, v_token, v_head;  // k_token, v_token: strides between blocks when paged
  void* out;
  long long out_token, out_head;
  int *err, *counters;
  float* partials;
  unsigned long long timeout_ns;
};

template <int D>
struct AttnCfg {
  static constexpr int HALVES = D / 64;
  static constexpr int TILE_BYTES = kAttnStep * D * 2;      // one k or v tile, or one row tile of q
  static constexpr int SLOTS = D == 128 ? 5 : 8;
  static constexpr int OFF_KV = 2 * TILE_BYTES;
  static constexpr int OFF_BAR = OFF_KV + SLOTS * TILE_BYTES;
  static constexpr int OFF_XCHG = TILE_BYTES;               // alt: the second row tile's place is free
  static constexpr int SMEM_BYTES = OFF_BAR + 3072;         // the ring begins on 1024 bytes (checked in the kernel)
  static constexpr int PART_ROWS = 256;
  static constexpr int PART_FLOATS = PART_ROWS * (D + 2);   // one partial slot: output, maxima, sums
};

enum AttnSite : int {
  SITE_ATTN_Q = 31, SITE_ATTN_Q_EMPTY, SITE_ATTN_KV_FULL, SITE_ATTN_KV_EMPTY, SITE_ATTN_S, SITE_ATTN_P, SITE_ATTN_PV,
  SITE_ATTN_XCHG, SITE_ATTN_DRAIN, SITE_ATTN_ALIGN
};

// ------------------------------------------------------------ tcgen05 forms
// K-major B tiles use make_sw128_desc.  v is the B operand of the second
// product with its rows (keys) along K: MN-major, 64 head elements (128 bytes)
// per row, eight-row groups 1024 bytes apart along K (stride byte offset), the
// next 64 elements of the head a whole [128 x 64] tile away (leading byte
// offset).
SVD_DEV uint64_t make_sw128_mn_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>((kAttnStep * 128) >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

constexpr uint32_t kIdescBMnMajor = 1u << 16;

// D[128 x N] (+)= A[128 x 16] B[16 x N], A in TMEM (two 16-bit elements per column).
SVD_DEV void umma_f16kind_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

SVD_DEV void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

SVD_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

SVD_DEV void tma_load_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

SVD_DEV void tma_load_4d_at(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

template <int N>
SVD_DEV void reg_alloc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
SVD_DEV void reg_dealloc() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

SVD_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
SVD_DEV uint32_t pack_pair(float lo, float hi);
template <>
SVD_DEV uint32_t pack_pair<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
SVD_DEV uint32_t pack_pair<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// --------------------------------------------------------------- the cutting
// sum over i < n of floor((a i + b) / m), a, b >= 0 (the Euclid-like floor sum).
SVD_DEV long long floor_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
  long long ans = 0;
  while (n > 0) {
    if (a >= m) {
      ans += (static_cast<long long>(n) * (n - 1) / 2) * (a / m);
      a %= m;
    }
    if (b >= m) {
      ans += static_cast<long long>(n) * (b / m);
      b %= m;
    }
    const unsigned long long y = static_cast<unsigned long long>(a) * n + b;
    if (y < m) break;
    n = static_cast<unsigned>(y / m);
    b = static_cast<unsigned>(y % m);
    const unsigned t = m;
    m = a;
    a = t;
  }
  return ans;
}

// One request as the kernel sees it, clipped to the tensors.
struct AttnSeq {
  int q0, n;     // first query row, queries
  int k0, m;     // first key row (packed), keys
  int first;     // keys that query -1 would see: m - n (causal), the context (tree)
};

SVD_DEV AttnSeq load_seq(const AttnParams& p, int b) {
  AttnSeq s;
  const int qa = p.cu_q[b], qb = p.cu_q[b + 1];
  s.q0 = min(max(qa, 0), p.q_tokens);
  s.n = max(min(qb, p.q_tokens) - s.q0, 0);
  if (p.lens != nullptr) {
    const int len = p.lens[b];
    s.k0 = 0;
    s.m = static_cast<int>(min(static_cast<long long>(max(len, 0)), static_cast<long long>(p.width) * p.block_size));
    s.first = len - (qb - qa);
  } else {
    const int ka = p.cu_k[b], kb = p.cu_k[b + 1];
    s.k0 = min(max(ka, 0), p.k_tokens);
    s.m = max(min(kb, p.k_tokens) - s.k0, 0);
    s.first = s.m - s.n;
  }
  return s;
}

SVD_DEV int unit_tokens(const AttnParams& p) { return p.alt ? p.tt : 2 * p.tt; }
// keys that the first t tokens of the request can see
SVD_DEV int keys_of(const AttnParams& p, const AttnSeq& s, int t) { return p.causal ? min(s.m, max(s.first + t, 0)) : s.m; }
SVD_DEV int steps_of(int keys) { return (keys + kAttnStep - 1) / kAttnStep; }
SVD_DEV int tiles_of(const AttnParams& p, const AttnSeq& s) { return (s.n + unit_tokens(p) - 1) / unit_tokens(p); }
// Steps of token tile i: at least one, so that rows which see no key are written too.
SVD_DEV int tile_steps(const AttnParams& p, const AttnSeq& s, int i) {
  return max(1, steps_of(keys_of(p, s, min((i + 1) * unit_tokens(p), s.n))));
}
// Steps of the tiles before tile i (i <= tiles).
SVD_DEV long long steps_before(const AttnParams& p, const AttnSeq& s, int i) {
  if (!p.causal) return static_cast<long long>(i) * max(1, steps_of(s.m));
  const int w = unit_tokens(p), tiles = tiles_of(p, s);
  long long sum = 0;
  if (i == tiles && i > 0) {  // the last tile may be cut short
    sum = tile_steps(p, s, i - 1);
    --i;
  }
  // tiles whose keys fit one step, then ceil((first + (k + 1) w) / step)
  const int room = kAttnStep - s.first;
  const int ones = min(i, room >= w ? room / w : 0);
  sum += ones;
  if (i > ones)
    sum += floor_sum(static_cast<unsigned>(i - ones), kAttnStep, static_cast<unsigned>(w),
                     static_cast<unsigned>(s.first + (ones + 1) * w + kAttnStep - 1));
  return sum;
}

// The segment of a unit that this CTA works on, and where the CTA goes next.
struct AttnWalk {
  AttnSeq s;
  int b, h, tile, tiles, j0, j1, steps;
  long long at, end;   // global step of the segment's first step; end of this CTA's piece

  SVD_DEV bool open(const AttnParams& p) {
    if (at >= end) return false;
    steps = tile_steps(p, s, tile);
    const long long left = end - at;
    j1 = left < steps - j0 ? j0 + static_cast<int>(left) : steps;
    return true;
  }
  SVD_DEV bool next(const AttnParams& p) {
    at += j1 - j0;
    if (at >= end) return false;
    j0 = 0;
    if (++tile == tiles) {
      tile = 0;
      if (++h == p.head_groups) {
        h = 0;
        do {
          if (++b >= p.batch) {
            at = end;
            return false;
          }
          s = load_seq(p, b);
        } while (s.n == 0);
        tiles = tiles_of(p, s);
      }
    }
    return open(p);
  }
  // rows of row tile i: first token, tokens, steps
  SVD_DEV int tile_t0(const AttnParams& p, int i) const { return tile * unit_tokens(p) + (p.alt ? 0 : i * p.tt); }
  SVD_DEV int tile_tokens(const AttnParams& p, int i) const { return max(0, min(p.tt, s.n - tile_t0(p, i))); }
  SVD_DEV int row_steps(const AttnParams& p, int i) const {
    const int nt = tile_tokens(p, i);
    return nt == 0 ? 0 : steps_of(keys_of(p, s, tile_t0(p, i) + nt));
  }
  // Whether softmax group i works on step j, and whether anything does.
  SVD_DEV bool active(const AttnParams& p, int i, int j, int steps_i) const {
    return j < steps_i && (!p.alt || ((j - j0) & 1) == i);
  }
};

// Places of the segment's tiles in the ring (loads since the segment began).
// pair: K0 V0 K1 V1 ...; alt: K0 K1 V0 K2 V1 ... (two score tiles in flight).
SVD_DEV int k_place(int alt, int i) { return !alt ? 2 * i : i == 0 ? 0 : 2 * i - 1; }
SVD_DEV int v_place(int alt, int i, int n) { return !alt ? 2 * i + 1 : i == n - 1 ? 2 * i + 1 : 2 * i + 2; }

// ------------------------------------------------------- the row-wise path
// The output of one row over the keys [j_lo, j_hi) of its segment, a warp per
// row, keys that the row does not see left out altogether.  Taken only where
// the tiled product gave a value that is not finite: the product multiplies
// every value in a tile, and 0 * inf in a masked place would reach rows that
// do not see it.  `base` is the row's maximum, in the exponent's units.
template <typename T, int D>
__device__ __noinline__ void attn_row(const AttnParams& p, const AttnSeq& s, int b, int token, int head, int kv_head,
                                      int j_lo, int j_hi, float base, float (&o)[D / 32]) {
  constexpr int E = D / 32;
  const int lane = lane_id();
  const T* q = static_cast<const T*>(p.q) + (s.q0 + token) * p.q_token + head * p.q_head;
  float qf[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qf[e] = elem_to_float(q[lane * E + e]);
    o[e] = 0.f;
  }
  const int sees = min(j_hi, p.causal ? s.first + token + 1 : s.m);
  const unsigned long long bits = p.mask != nullptr ? p.mask[s.q0 + token] : 0;
  const float c = p.neg ? -p.c : p.c;
  for (int j = j_lo; j < sees; ++j) {
    const T *kr, *vr;
    if (p.lens != nullptr) {
      const int node = j - s.first;
      if (node >= 0 && (p.mask != nullptr ? node >= 64 || !(bits >> node & 1) : node > token)) continue;
      const int page = p.table[b * p.ld_table + (j >> p.block_shift)];
      if (page < 0 || page >= p.num_blocks) continue;
      const long long in = (kv_head * static_cast<long long>(p.block_size) + (j & (p.block_size - 1))) * D;
      kr = static_cast<const T*>(p.k) + page * p.k_token + in;
      vr = static_cast<const T*>(p.v) + page * p.v_token + in;
    } else {
      kr = static_cast<const T*>(p.k) + (s.k0 + j) * p.k_token + kv_head * p.k_head;
      vr = static_cast<const T*>(p.v) + (s.k0 + j) * p.v_token + kv_head * p.v_head;
    }
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) dot += qf[e] * elem_to_float(kr[lane * E + e]);
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float w = exp2f(dot * c - base);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += w * elem_to_float(vr[lane * E + e]);
  }
}

// -------------------------------------------------------------- the kernel
struct AttnShared {
  uint64_t q_full, q_empty, xchg, drain;
  uint64_t s_full[2], p_ready[2], pv_done[2];
  uint64_t kv_full[8], kv_empty[8];
  uint32_t tmem;
  int abort_flag, last;
  int start_b, start_h, start_tile, start_j;
  long long start, end, total, per;
  long long scan[kAttnThreads / 32];
  float m[256], l[256];         // joining: per-row maximum and 1 / sum
};

// mbar_wait by a whole warp: every lane gets the same answer, so that no lane
// is left alone at a warp-wide instruction.
SVD_DEV bool warp_wait(uint64_t* bar, uint32_t parity, const WaitCtx& ctx, int site, bool honour_abort = true) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, ctx, site, honour_abort));
}

// Every CTA finds its piece of the line of steps.
SVD_DEV void find_piece(const AttnParams& p, AttnShared* sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int NW = kAttnThreads / 32;
  long long base = 0, total = 0;
  // first the total, then (second round) the request that holds the piece's first step
  for (int round = 0; round < 2; ++round) {
    base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kAttnThreads) {
      const int b = b0 + tid;
      long long mine = 0, unit = 0;
      AttnSeq s{};
      if (b < p.batch) {
        s = load_seq(p, b);
        unit = s.n > 0 ? steps_before(p, s, tiles_of(p, s)) : 0;
        mine = unit * p.head_groups;
      }
      long long inc = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      if (lane == 31) sh->scan[warp] = inc;
      __syncthreads();
      long long before = base, all = 0;
      for (int w = 0; w < NW; ++w) {
        if (w < warp) before += sh->scan[w];
        all += sh->scan[w];
      }
      before += inc - mine;
      __syncthreads();
      base += all;
      if (p.batch <= kAttnThreads) total = base;  // one chunk: the total is known at once
      if (round == 1 || p.batch <= kAttnThreads) {
        const long long per = max(static_cast<long long>(p.min_steps), (total + gridDim.x - 1) / gridDim.x);
        const long long start = per * blockIdx.x;
        if (tid == 0) {
          sh->per = per;
          sh->start = start;
          sh->end = min(start + per, total);
        }
        if (start >= before && start < before + mine) {
          const long long in = start - before;
          sh->start_b = b;
          sh->start_h = static_cast<int>(in / unit);
          const long long rem = in - (in / unit) * unit;
          int lo = 0, hi = tiles_of(p, s);  // the last tile with at most rem steps before it
          while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (steps_before(p, s, mid) <= rem) lo = mid;
            else hi = mid;
          }
          sh->start_tile = lo;
          sh->start_j = static_cast<int>(rem - steps_before(p, s, lo));
        }
      }
    }
    total = base;
    if (p.batch <= kAttnThreads) break;
  }
}

SVD_DEV AttnWalk first_walk(const AttnParams& p, const AttnShared* sh) {
  AttnWalk w{};
  w.at = sh->start;
  w.end = sh->end;
  if (w.at < w.end) {
    w.b = sh->start_b;
    w.h = sh->start_h;
    w.tile = sh->start_tile;
    w.j0 = sh->start_j;
    w.s = load_seq(p, w.b);
    w.tiles = tiles_of(p, w.s);
  }
  return w;
}

template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(kAttnThreads, 1)
    attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p) {
  using Cfg = AttnCfg<D>;
  constexpr bool F16 = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t smem[];
  AttnShared* sh = reinterpret_cast<AttnShared*>(smem + Cfg::OFF_BAR);
  static_assert(Cfg::OFF_BAR + sizeof(AttnShared) <= Cfg::SMEM_BYTES && Cfg::SMEM_BYTES <= 232448, "shared memory");
  if ((smem_addr(smem) & 1023u) != 0) {  // the swizzle counts from 1024-byte boundaries
    if (threadIdx.x == 0) atomicCAS(p.err, 0, SITE_ATTN_ALIGN);
    return;
  }
  const int warp = threadIdx.x >> 5;
  const int lane = static_cast<int>(lane_id());

  if (threadIdx.x == 0) {
    mbar_init(&sh->q_full, 1);
    mbar_init(&sh->q_empty, 1);
    mbar_init(&sh->xchg, 256);
    mbar_init(&sh->drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->p_ready[i], 128);
      mbar_init(&sh->pv_done[i], 1);
    }
    for (int i = 0; i < Cfg::SLOTS; ++i) {
      mbar_init(&sh->kv_full[i], 1);
      mbar_init(&sh->kv_empty[i], 1);
    }
    sh->abort_flag = 0;
    fence_mbarrier_init();
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 8) {
    tmem_alloc(&sh->tmem, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  find_piece(p, sh);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;
  const WaitCtx ctx{&sh->abort_flag, p.err, p.timeout_ns};
  AttnWalk w = first_walk(p, sh);

  // rows of no request give zeros
  {
    const int lo = min(max(p.cu_q[0], 0), p.q_tokens), hi = min(max(p.cu_q[p.batch], lo), p.q_tokens);
    const int heads = p.head_groups * p.gp;
    const long long rows = static_cast<long long>(lo + p.q_tokens - hi) * heads;
    for (long long r = blockIdx.x * static_cast<long long>(kAttnThreads) + threadIdx.x; r < rows;
         r += static_cast<long long>(gridDim.x) * kAttnThreads) {
      const int t = static_cast<int>(r / heads), h = static_cast<int>(r % heads);
      T* dst = static_cast<T*>(p.out) + static_cast<long long>(t < lo ? t : t - lo + hi) * p.out_token + h * p.out_head;
      for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
    }
  }

  if (warp >= 8) {
    reg_dealloc<88>();
    if (warp == 9) {
      // ------------------------------------------------------------ TMA warp
      int ld = 0, seg = 0;
      bool ok = true;
      const int q_rows = p.tt * p.gp;
      const uint32_t tile_bytes = Cfg::TILE_BYTES;
      for (bool more = w.open(p); more && ok; more = w.next(p), ++seg) {
        if (!warp_wait(&sh->q_empty, (seg & 1) ^ 1, ctx, SITE_ATTN_Q_EMPTY)) break;
        if (lane == 0) {
          const int qt = p.alt ? 1 : 2;
          mbar_arrive_expect_tx(&sh->q_full, static_cast<uint32_t>(qt * Cfg::HALVES * q_rows * 128));
          for (int i = 0; i < qt; ++i)
            for (int hf = 0; hf < Cfg::HALVES; ++hf)
              tma_load_4d_at(&map_q, &sh->q_full, smem + i * Cfg::TILE_BYTES + hf * (kAttnStep * 128), hf * 64, 0, w.h,
                             w.s.q0 + w.tile_t0(p, i));
        }
        const int kv_head = w.h * p.gp / p.group;
        const int n = w.j1 - w.j0;
        // one tile of k or v into the next slot of the ring
        const auto load = [&](const CUtensorMap* map, int j) -> bool {
          const int slot = ld % Cfg::SLOTS;
          if (!warp_wait(&sh->kv_empty[slot], static_cast<uint32_t>(ld / Cfg::SLOTS & 1) ^ 1u, ctx, SITE_ATTN_KV_EMPTY))
            return false;
          ++ld;
          uint8_t* dst = smem + Cfg::OFF_KV + slot * Cfg::TILE_BYTES;
          if (lane == 0) mbar_arrive_expect_tx(&sh->kv_full[slot], tile_bytes);
          __syncwarp();
          if constexpr (PAGED) {
            // a lane per block; a block the table does not name is read out of range, as zeros
            const int rows = min(p.block_size, kAttnStep);
            if (lane * rows < kAttnStep) {
              const int key = j * kAttnStep + lane * rows;
              const int entry = key >> p.block_shift;
              int page = -1;
              if (key < w.s.m) page = p.table[w.b * p.ld_table + entry];
              if (page < 0 || page >= p.num_blocks) page = p.num_blocks;
              for (int hf = 0; hf < Cfg::HALVES; ++hf)
                tma_load_4d_at(map, &sh->kv_full[slot], dst + hf * (kAttnStep * 128) + lane * rows * 128, hf * 64,
                               key & (p.block_size - 1), kv_head, page);
            }
          } else {
            if (lane == 0)
              for (int hf = 0; hf < Cfg::HALVES; ++hf)
                tma_load_3d(map, &sh->kv_full[slot], dst + hf * (kAttnStep * 128), hf * 64, kv_head,
                            w.s.k0 + j * kAttnStep);
          }
          return true;
        };
        if (!p.alt) {
          for (int i = 0; i < n && ok; ++i) ok = load(&map_k, w.j0 + i) && load(&map_v, w.j0 + i);
        } else {
          ok = load(&map_k, w.j0);
          for (int i = 0; i < n && ok; ++i) {
            if (i + 1 < n) ok = load(&map_k, w.j0 + i + 1);
            ok = ok && load(&map_v, w.j0 + i);
          }
        }
      }
      // every load in flight has landed before the CTA ends
      for (int sl = 0; sl < Cfg::SLOTS; ++sl)
        if (ld > sl) {
          const int last = sl + (ld - 1 - sl) / Cfg::SLOTS * Cfg::SLOTS;
          mbar_wait(&sh->kv_full[sl], static_cast<uint32_t>(last / Cfg::SLOTS & 1), ctx, SITE_ATTN_DRAIN, false);
        }
      if (seg > 0) mbar_wait(&sh->q_full, static_cast<uint32_t>((seg - 1) & 1), ctx, SITE_ATTN_DRAIN, false);
    } else if (warp == 8) {
      // ------------------------------------------------------------ MMA warp
      constexpr uint32_t idesc_s = make_idesc_16bit(128, kAttnStep, F16);
      constexpr uint32_t idesc_o = make_idesc_16bit(128, D, F16) | kIdescBMnMajor;
      int ld = 0, seg = 0;
      int n_p[2] = {0, 0};  // probability tiles consumed, per group
      bool ok = true;
      const auto slot_of = [&](int place) { return (ld + place) % Cfg::SLOTS; };
      const auto wait_full = [&](int place) {
        const int x = ld + place;
        return warp_wait(&sh->kv_full[x % Cfg::SLOTS], static_cast<uint32_t>(x / Cfg::SLOTS & 1), ctx, SITE_ATTN_KV_FULL);
      };
      const auto release = [&](int place) {
        if (lane == 0) umma_commit(&sh->kv_empty[slot_of(place)]);
      };
      const auto scores = [&](int i, int place) {  // S_i = Q_i K^T
        if (lane == 0) {
          const uint32_t a = smem_addr(smem + (p.alt ? 0 : i) * Cfg::TILE_BYTES);
          const uint32_t bk = smem_addr(smem + Cfg::OFF_KV + slot_of(place) * Cfg::TILE_BYTES);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k / 4) * (kAttnStep * 128) + (k % 4) * 32;
            umma_f16kind(tmem + i * 128, make_sw128_desc(a + off), make_sw128_desc(bk + off), idesc_s, k > 0);
          }
          umma_commit(&sh->s_full[i]);
        }
      };
      const auto values = [&](int i, int place, bool first) {  // O_i (+)= P_i V
        if (lane == 0) {
          const uint32_t bv = smem_addr(smem + Cfg::OFF_KV + slot_of(place) * Cfg::TILE_BYTES);
#pragma unroll
          for (int k = 0; k < kAttnStep / 16; ++k)
            umma_f16kind_ts(tmem + 256 + i * D, tmem + i * 128 + k * 8, make_sw128_mn_desc(bv + k * 2048), idesc_o,
                            !first || k > 0);
          umma_commit(&sh->pv_done[i]);
        }
      };
      // v rows behind the last key are other requests' or nobody's: zeros
      const auto clean = [&](int place, int j) {
        const int valid = w.s.m - j * kAttnStep;
        if (valid < kAttnStep) {
          uint8_t* t = smem + Cfg::OFF_KV + slot_of(place) * Cfg::TILE_BYTES;
          for (int x = max(valid, 0) * 8 + lane; x < kAttnStep * 8; x += 32)
            for (int hf = 0; hf < Cfg::HALVES; ++hf)
              *reinterpret_cast<uint4*>(t + hf * (kAttnStep * 128) + x * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
      };
      for (bool more = w.open(p); more && ok; more = w.next(p), ++seg) {
        const int n = w.j1 - w.j0;
        const int st[2] = {w.row_steps(p, 0), w.row_steps(p, 1)};
        const int last_place = 2 * n;
        bool started[2] = {false, false};
        ok = warp_wait(&sh->q_full, seg & 1, ctx, SITE_ATTN_Q);
        if (!ok) break;
        tc_fence_after();
        // the first score tiles
        for (int x = 0; x < (p.alt ? min(n, 2) : 1) && ok; ++x) {
          const int pl = k_place(p.alt, x);
          ok = wait_full(pl);
          if (!ok) break;
          tc_fence_after();
          for (int i = 0; i < 2; ++i)
            if (w.active(p, i, w.j0 + x, st[i])) scores(i, pl);
          release(pl);
        }
        const int ahead = p.alt ? 2 : 1;
        for (int x = 0; x < n && ok; ++x) {
          const int j = w.j0 + x;
          const int pv = v_place(p.alt, x, n), pk = k_place(p.alt, x + ahead);
          const bool more_k = x + ahead < n;
          bool have_v = false, have_k = false;
          for (int i = 0; i < 2 && ok; ++i) {
            if (w.active(p, i, j, st[i])) {
              ok = warp_wait(&sh->p_ready[i], n_p[i] & 1, ctx, SITE_ATTN_P);
              if (!ok) break;
              ++n_p[i];
              if (!have_v) {
                ok = wait_full(pv);
                if (!ok) break;
                clean(pv, j);
                have_v = true;
              }
              tc_fence_after();
              values(i, pv, !started[i]);
              started[i] = true;
            }
            if (more_k && w.active(p, i, j + ahead, st[i])) {
              if (!have_k) {
                ok = wait_full(pk);
                if (!ok) break;
                have_k = true;
              }
              tc_fence_after();
              scores(i, pk);
            }
          }
          if (!ok) break;
          // a tile that nothing used has landed before its slot is handed back
          if (!have_v) ok = wait_full(pv);
          if (ok && more_k && !have_k) ok = wait_full(pk);
          if (!ok) break;
          release(pv);
          if (more_k) release(pk);
        }
        if (!ok) break;
        if (lane == 0) umma_commit(&sh->q_empty);
        ld += last_place;
      }
      if (lane == 0) umma_commit(&sh->drain);
      __syncwarp();
      mbar_wait(&sh->drain, 0, ctx, SITE_ATTN_DRAIN, false);
    }
  } else {
    // -------------------------------------------------------- softmax groups
    reg_alloc<208>();
    const int i = warp >> 2;                          // group
    const int r = threadIdx.x & 127;                  // row of the tile, lane of TMEM
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + i * 128, t_o = tmem + lanes + 256 + i * D;
    const int row_token = r / p.gp, row_head = r - row_token * p.gp;
    int n_s = 0, n_x = 0;                             // score tiles taken; exchanges
    bool ok = true;
    const auto meet = [&]() {                         // all 256 softmax threads
      mbar_arrive(&sh->xchg);
      const bool k = warp_wait(&sh->xchg, n_x & 1, ctx, SITE_ATTN_XCHG);
      ++n_x;
      return k;
    };
    for (bool more = w.open(p); more; more = w.next(p)) {
      const int steps_i = w.row_steps(p, i);
      const int t0 = w.tile_t0(p, i), token = t0 + row_token;
      const bool row_ok = row_token < w.tile_tokens(p, i);
      // keys below `open` are seen by every row of the tile, keys from `sees` on by none of this row (outside a mask)
      const int open = p.tree ? w.s.first : p.causal ? w.s.first + t0 + 1 : w.s.m;
      const int sees = p.tree ? (p.mask != nullptr ? min(w.s.first, w.s.m) : min(w.s.first + token + 1, w.s.m))
                              : p.causal ? min(w.s.first + token + 1, w.s.m) : w.s.m;
      const unsigned long long bits = p.mask != nullptr && row_ok ? p.mask[w.s.q0 + token] : 0;
      float m = -INFINITY, l = 0.f;                   // m in units of the scores
      bool some = false;
      const int stride = p.alt ? 2 : 1;
      const int first_j = w.j0 + (p.alt ? i : 0), last_j = min(w.j1, steps_i);
      for (int j = first_j; j < last_j; j += stride) {
        unsigned bad_pages = 0;
        if constexpr (PAGED) {
          const int rows = min(p.block_size, kAttnStep);
          const int key = j * kAttnStep + lane * rows;
          bool bad = false;
          if (lane * rows < kAttnStep && key < w.s.m) {
            const int page = p.table[w.b * p.ld_table + (key >> p.block_shift)];
            bad = page < 0 || page >= p.num_blocks;
          }
          bad_pages = __ballot_sync(0xffffffffu, bad);
        }
        if (!(ok = warp_wait(&sh->s_full[i], n_s & 1, ctx, SITE_ATTN_S))) break;
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int x = 0; x < 4; ++x) tmem_ld_x32(t_s + x * 32, reinterpret_cast<uint32_t(&)[32]>(s[x * 32]));
        tmem_ld_wait();
        if (p.neg) {
#pragma unroll
          for (int x = 0; x < 128; ++x) s[x] = -s[x];
        }
        const int rel = j * kAttnStep;
        if (rel + kAttnStep > min(open, w.s.m) || bad_pages != 0) {
          // one bit per key of the step
          uint32_t vis[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int lim = sees - rel - 32 * x;
            vis[x] = lim >= 32 ? 0xffffffffu : lim > 0 ? (1u << lim) - 1u : 0u;
          }
          if (p.mask != nullptr) {
            // the tree's 64 bits, moved to where its first key lies in this step
            const int at = w.s.first - rel;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int sh_by = at - 32 * x;          // bit 0 of the tree in this word's coordinates
              uint32_t part = 0;
              if (sh_by > -64 && sh_by < 32)
                part = sh_by >= 0 ? static_cast<uint32_t>(bits << sh_by) : static_cast<uint32_t>(bits >> -sh_by);
              const int end = w.s.m - rel - 32 * x;   // keys that exist
              part &= end >= 32 ? 0xffffffffu : end > 0 ? (1u << end) - 1u : 0u;
              vis[x] |= part;
            }
          }
          if constexpr (PAGED) {
            if (bad_pages != 0) {
              const int rows = min(p.block_size, kAttnStep);
              for (unsigned rest = bad_pages; rest != 0; rest &= rest - 1) {
                const int lo = (__ffs(rest) - 1) * rows;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const int a = max(lo - 32 * x, 0), z = min(lo + rows - 32 * x, 32);
                  if (a < z) vis[x] &= ~((z - a == 32 ? 0xffffffffu : (1u << (z - a)) - 1u) << a);
                }
              }
            }
          }
#pragma unroll
          for (int x = 0; x < 128; ++x)
            if (!(vis[x / 32] >> (x % 32) & 1u)) s[x] = -INFINITY;
        }
        float top = fmaxf(s[0], s[1]), top2 = fmaxf(s[2], s[3]);
#pragma unroll
        for (int x = 4; x < 128; x += 4) {
          top = fmaxf(top, fmaxf(s[x], s[x + 1]));
          top2 = fmaxf(top2, fmaxf(s[x + 2], s[x + 3]));
        }
        top = fmaxf(top, top2);
        // a new base only where the maximum has grown by more than the stale one absorbs
        const bool grow = top > m && (m == -INFINITY || (top - m) * p.c > kAttnLazy);
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? exp2_approx((m - top) * p.c) : 1.0f;
          if (grow) {
            m = top;
            l *= alpha;
          }
          if (some) {
            if (!(ok = warp_wait(&sh->pv_done[i], (n_s - 1) & 1, ctx, SITE_ATTN_PV))) break;
            tc_fence_after();
#pragma unroll 1
            for (int x = 0; x < D; x += 32) {
              uint32_t o[32];
              tmem_ld_x32(t_o + x, o);
              tmem_ld_wait();
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha);
              tmem_st_x32(t_o + x, o);
            }
            tmem_st_wait();
          }
        }
        const float base = m == -INFINITY ? 0.f : m * p.c;
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t pk[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            const float a = exp2_approx(fmaf(s[hf * 64 + 2 * x], p.c, -base));
            const float b = exp2_approx(fmaf(s[hf * 64 + 2 * x + 1], p.c, -base));
            sum0 += a;
            sum1 += b;
            pk[x] = pack_pair<T>(a, b);
          }
          tmem_st_x32(t_s + hf * 32, pk);
        }
        l += sum0 + sum1;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sh->p_ready[i]);
        ++n_s;
        some = true;
      }
      ok = __all_sync(0xffffffffu, ok && *ctx.abort_flag == 0);
      if (!ok) break;
      if (some) {
        if (!(ok = warp_wait(&sh->pv_done[i], (n_s - 1) & 1, ctx, SITE_ATTN_PV))) break;
        tc_fence_after();
      }
      // ---------------------------------------------------- the segment's end
      const bool whole = w.j0 == 0 && w.j1 == w.steps;
      float m_out = m == -INFINITY ? -INFINITY : m * p.c, l_out = l;
      float w0 = 1.f, w1 = 0.f;                       // alt: weights of the groups' outputs
      bool has0 = some, has1 = false;
      if (p.alt) {
        float* x = reinterpret_cast<float*>(smem + Cfg::OFF_XCHG);
        x[i * 128 + r] = m_out;
        x[256 + i * 128 + r] = l;
        if (!(ok = meet())) break;
        tc_fence_after();
        const float m0 = x[r], m1 = x[128 + r];
        const float l0 = x[256 + r], l1 = x[384 + r];
        has0 = true;                                  // the first step is group 0's
        has1 = w.j1 - w.j0 > 1;
        if (steps_i <= w.j0) has0 = has1 = false;     // no key at all
        m_out = fmaxf(m0, m1);
        const float safe = m_out == -INFINITY ? 0.f : m_out;
        w0 = exp2_approx(m0 - safe);
        w1 = exp2_approx(m1 - safe);
        l_out = l0 * w0 + l1 * w1;
      }
      const int c_lo = p.alt ? i * (D / 2) : 0, c_hi = p.alt ? c_lo + D / 2 : D;
      const float inv = l_out == 0.f ? 0.f : 1.f / l_out;
      const int row = (p.alt ? 0 : i * 128) + r;
      const int head = w.h * p.gp + row_head, kv_head = w.h * p.gp / p.group;
      float* part = nullptr;
      long long unit0 = w.at - w.j0;
      if (!whole)
        part = p.partials + (static_cast<long long>(blockIdx.x) * 2 + (w.at == sh->start ? 0 : 1)) * Cfg::PART_FLOATS;
      T* dst = static_cast<T*>(p.out) + static_cast<long long>(w.s.q0 + token) * p.out_token + head * p.out_head;
      float probe = 0.f;                              // NaN when any output is not finite
#pragma unroll 1
      for (int x = c_lo; x < c_hi; x += 32) {
        float v[32];
        if (p.alt) {
          uint32_t o0[32], o1[32];
          tmem_ld_x32(tmem + lanes + 256 + x, o0);
          tmem_ld_x32(tmem + lanes + 256 + D + x, o1);
          tmem_ld_wait();
#pragma unroll
          for (int y = 0; y < 32; ++y)
            v[y] = (has0 ? w0 * __uint_as_float(o0[y]) : 0.f) + (has1 ? w1 * __uint_as_float(o1[y]) : 0.f);
        } else {
          tmem_ld_x32(t_o + x, reinterpret_cast<uint32_t(&)[32]>(v));
          tmem_ld_wait();
          if (!has0) {
#pragma unroll
            for (int y = 0; y < 32; ++y) v[y] = 0.f;
          }
        }
#pragma unroll
        for (int y = 0; y < 32; ++y) probe = fmaf(v[y], 0.f, probe);
        if (row_ok) {
          if (whole) {
#pragma unroll
            for (int y = 0; y < 32; y += 8) {
              uint4 o;
              o.x = pack_pair<T>(v[y] * inv, v[y + 1] * inv);
              o.y = pack_pair<T>(v[y + 2] * inv, v[y + 3] * inv);
              o.z = pack_pair<T>(v[y + 4] * inv, v[y + 5] * inv);
              o.w = pack_pair<T>(v[y + 6] * inv, v[y + 7] * inv);
              *reinterpret_cast<uint4*>(dst + x + y) = o;
            }
          } else {
#pragma unroll
            for (int y = 0; y < 32; y += 4)
              __stcg(reinterpret_cast<float4*>(part) + ((x + y) >> 2) * Cfg::PART_ROWS + row,
                     make_float4(v[y], v[y + 1], v[y + 2], v[y + 3]));
          }
        }
      }
      if (!whole && row_ok && c_lo == 0) {
        __stcg(part + Cfg::PART_ROWS * D + row, m_out);
        __stcg(part + Cfg::PART_ROWS * (D + 1) + row, l_out);
      }
      // rows that a masked place may have reached: over again, key by key
      unsigned redo = __ballot_sync(0xffffffffu, row_ok && probe != 0.f);
      while (redo != 0) {
        const int src = __ffs(redo) - 1;
        redo &= redo - 1;
        const int tk = __shfl_sync(0xffffffffu, token, src), hd = __shfl_sync(0xffffffffu, head, src);
        const int rw = __shfl_sync(0xffffffffu, row, src);
        const float bs = __shfl_sync(0xffffffffu, m_out == -INFINITY ? 0.f : m_out, src);
        const float iv = __shfl_sync(0xffffffffu, inv, src);
        float o[D / 32];
        attn_row<T, D>(p, w.s, w.b, tk, hd, kv_head, w.j0 * kAttnStep, min(w.j1 * kAttnStep, w.s.m), bs, o);
        __syncwarp();
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          const int d = lane * (D / 32) + e;
          if (d >= c_lo && d < c_hi) {
            if (whole)
              static_cast<T*>(p.out)[static_cast<long long>(w.s.q0 + tk) * p.out_token + hd * p.out_head + d] =
                  elem_from_float<T>(o[e] * iv);
            else
              __stcg(part + ((d >> 2) * Cfg::PART_ROWS + rw) * 4 + (d & 3), o[e]);
          }
        }
      }
      if (p.alt) {
        // both groups have read both outputs before either writes new ones
        tc_fence_before();
        if (!(ok = meet())) break;
      }
      if (!whole) {
        // the last CTA of the unit to arrive joins the partials, in the order of the keys
        __threadfence();
        if (!(ok = meet())) break;
        const int c0 = static_cast<int>(unit0 / sh->per), c1 = static_cast<int>((unit0 + w.steps - 1) / sh->per);
        if (threadIdx.x == 0) {
          const int arrived = atom_add_acq_rel_gpu(&p.counters[c0], 1);
          sh->last = arrived == c1 - c0;
          if (sh->last) p.counters[c0] = 0;
        }
        if (!(ok = meet())) break;
        if (sh->last) {
          __threadfence();
          const int tid = threadIdx.x;
          const long long first_slot = (unit0 == static_cast<long long>(c0) * sh->per) ? 2LL * c0 : 2LL * c0 + 1;
          const auto slot = [&](int cta) -> const float* {
            return p.partials + (cta == c0 ? first_slot : 2LL * cta) * Cfg::PART_FLOATS;
          };
          const int tok0 = w.tile_tokens(p, 0), tok1 = p.alt ? 0 : w.tile_tokens(p, 1);
          // per row: the common maximum and 1 / sum
          {
            const int rr = tid;                       // row of the unit
            const bool there = (rr & 127) / p.gp < (rr < 128 ? tok0 : tok1);
            float mm = -INFINITY, ll = 0.f;
            if (there) {
              for (int cta = c0; cta <= c1; ++cta) mm = fmaxf(mm, __ldcg(slot(cta) + Cfg::PART_ROWS * D + rr));
              const float safe = mm == -INFINITY ? 0.f : mm;
              for (int cta = c0; cta <= c1; ++cta)
                ll += exp2_approx(__ldcg(slot(cta) + Cfg::PART_ROWS * D + rr) - safe) *
                      __ldcg(slot(cta) + Cfg::PART_ROWS * (D + 1) + rr);
              mm = safe;
            }
            sh->m[rr] = mm;
            sh->l[rr] = ll == 0.f ? 0.f : 1.f / ll;
          }
          if (!(ok = meet())) break;
          const int rows0 = tok0 * p.gp, rows = rows0 + tok1 * p.gp;
          const int items = rows * (D / 4);
          constexpr int U = 4;
          for (int it0 = tid; it0 < items; it0 += 256 * U) {
            float4 acc[U];
            int rowu[U], du[U];
            float mu[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int it = min(it0 + 256 * u, items - 1);
              du[u] = it / rows;
              const int x = it - du[u] * rows;
              rowu[u] = x < rows0 ? x : 128 + x - rows0;
              mu[u] = sh->m[rowu[u]];
              acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            for (int cta = c0; cta <= c1; ++cta) {
              const float* sl = slot(cta);
              float wt[U];
              float4 o[U];
#pragma unroll
              for (int u = 0; u < U; ++u) {
                wt[u] = __ldcg(sl + Cfg::PART_ROWS * D + rowu[u]);
                o[u] = __ldcg(reinterpret_cast<const float4*>(sl) + du[u] * Cfg::PART_ROWS + rowu[u]);
              }
#pragma unroll
              for (int u = 0; u < U; ++u) {
                const float f = exp2_approx(wt[u] - mu[u]);
                acc[u].x = fmaf(f, o[u].x, acc[u].x);
                acc[u].y = fmaf(f, o[u].y, acc[u].y);
                acc[u].z = fmaf(f, o[u].z, acc[u].z);
                acc[u].w = fmaf(f, o[u].w, acc[u].w);
              }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
              if (it0 + 256 * u < items) {
                const int rr = rowu[u] & 127, tl = rowu[u] >> 7;
                const float iv = sh->l[rowu[u]];
                const int tk = w.tile_t0(p, tl) + rr / p.gp, hd = w.h * p.gp + rr % p.gp;
                uint2 o;
                o.x = pack_pair<T>(acc[u].x * iv, acc[u].y * iv);
                o.y = pack_pair<T>(acc[u].z * iv, acc[u].w * iv);
                *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + static_cast<long long>(w.s.q0 + tk) * p.out_token +
                                          hd * p.out_head + du[u] * 4) = o;
              }
            }
          }
          if (!(ok = meet())) break;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace svdmlp
