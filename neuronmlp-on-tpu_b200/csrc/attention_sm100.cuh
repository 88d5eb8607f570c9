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
// Two schedules (PAIR, chosen by the host).  A unit is one (request, head
// group, token tile).  PAIR: a unit has two row tiles, which share every k and
// v tile, 128 keys per step; for requests of more than 128 rows.  Otherwise a
// unit has one row tile, 64 keys per step, and the CTA holds two independent
// workers, each with its own ring, MMA warp and TMA warp, so that one's loads
// and epilogues lie beside the other's products: a second row tile would be
// empty, and the bytes of k and v bound.
//
// Work.  The steps of all units, and a few steps' worth for every unit's
// beginning and end, form one line, cut into equal pieces, one per
// worker (persistent, one CTA per SM): every CTA computes its cuts itself from
// the request lengths on the device, so ragged lengths, long prompts and a
// single long context load every SM alike.  A cut inside a short unit moves to
// its nearer end (always to its start: 39 instead of 33 us for 4 requests of up
// to 512 tokens behind 2000 keys).  A unit that a cut divides leaves fp32
// partials (maximum, sum, unnormalised output) in the workspace, and the worker
// that begins it a note of where they are; a second kernel joins them, in the
// order of the keys.
// (Joined by the worker that arrives last instead, a CTA read up to a megabyte
// on its own: one request of 16 drafted tokens on 8000 keys 52 us, 25 us with
// the second kernel; 8 requests of one token on 2000 keys 31 and 21 us.)
//
// Roles (384 threads): two softmax warpgroups, one thread per row; an MMA and a
// TMA warp per worker.  TMEM (512 columns): per group 128 columns of scores and
// one output tile.  The probabilities overwrite the scores as 16-bit pairs and
// are the A operand of the second product.  With 64-key steps the 128 columns
// are two score tiles, and the scores run two steps ahead: the MMA warp issues
// P V(j) and then Q K(j + 2), which takes P(j)'s place, while the group already
// works on the scores of step j + 1, across the ends of units too.  PAIR has one
// tile of 128 keys per group, one step ahead, and the two groups take turns on
// the tensor pipe and on the exponential unit; P V starts on the first 64 keys
// while the exponentials of the others are computed.  (With two tiles of 64 the
// issue of the products bounds PAIR, with or without a softmax: 565 us where
// this took 490, a few calls at a time, at one prompt of 8192 tokens, 32 and 8
// heads of 128.)  The
// output is rescaled only when a row's maximum grows by more than 8 (in powers of
// two): a stale base keeps probabilities below 2^8, which the 16-bit types and
// the fp32 sums hold without loss.
//
// What bounds it.  Long prompts: per 128 keys and 128 rows at head_dim 128 the
// tensor pipe takes 1100 cycles and the exponential unit 1024, and the chain
// scores -> maximum -> exponentials -> P V -> scores of a tile some 3000, so that
// two tiles in turn leave gaps in both (without the softmax's arithmetic the
// same products took 395 instead of 490 us); 513 us for a call after a pause over
// other inputs, 545 to 565 in calls that follow one another for long, where the
// power limit takes the clock down.  The PAIR kernels spill some 300 bytes a
// thread around the softmax (168 registers at launch).  Few rows on many
// keys: the bytes of k and v, read once; for short calls the start of the CTAs
// (the cuts 2 to 4 us, block tables and first loads 3) and the join.  One token on
// 65537 keys: 54 us, 5.1 TB/s, and 5 us for the join.
#pragma once

#include <climits>
#include <type_traits>

#include "attention_line.h"
#include "rope_pages.cuh"

namespace svdmlp {

constexpr int kAttnThreads = 384;
constexpr int kAttnMaxGrid = 512;     // CTAs that the workspace has room for
constexpr float kAttnLazy = 8.0f;     // growth of the maximum (log2) that a stale base absorbs

// What a worker leaves for the join: the unit that it begins and does not
// finish.  Its partials are this worker's second one and the first ones of the
// `more` workers after it.
struct AttnSplit {
  int more;             // 0: none
  int rows0, rows;      // rows of the first row tile, of the unit
  int token0, head0;    // first query row (in the tensor) and head
  int pad[3];
};

struct AttnParams {
  int batch, q_tokens, k_tokens;
  int head_groups, gp, group;         // units per token tile; query heads per unit; query heads per kv head
  int tt, causal, tree;
  int snap;                           // units of up to this many steps are not divided
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
  int* err;
  float* partials;
  AttnSplit* splits;           // per worker
  unsigned long long timeout_ns;
};

template <int D, bool PAIR>
struct AttnCfg {
  static constexpr int HALVES = D / 64;
  static constexpr int WORKERS = PAIR ? 1 : 2;              // per CTA
  static constexpr int USERS = PAIR ? 2 : 1;                // MMA warps per worker, one per row tile
  // Registers of a softmax thread and of the other warps, when moved between
  // them (three warps share a partition's 16 K: 168 each at launch).  PAIR holds
  // 128 scores a thread; with 64 the softmax fits in 168, and the MMA and TMA
  // warps run without spills (measured: 65 K decoding 66 -> 58 us).
  static constexpr int SOFTMAX_REGS = 200, OTHER_REGS = 104;
  static constexpr int Q_BYTES = 128 * D * 2;               // one row tile of q
  static constexpr int STEP = PAIR ? 128 : 64;              // keys per step
  static constexpr int SLOT_BYTES = STEP * D * 2;           // k or v of one step
  static constexpr int HALF_BYTES = STEP * 128;             // 64 elements of the head for every key of a slot
  static constexpr int SLOTS = D == 128 ? 5 : 8;            // per worker
  static constexpr int TILES = 128 / STEP;                  // score tiles per group: steps that the scores run ahead
  static constexpr int OFF_KV = 2 * Q_BYTES;
  static constexpr int OFF_BAR = OFF_KV + WORKERS * SLOTS * SLOT_BYTES;
  static constexpr int SMEM_BYTES = OFF_BAR + 3072;         // the ring begins on 1024 bytes (checked in the kernel)
  static constexpr int PART_ROWS = PAIR ? 256 : 128;
  static constexpr int PART_FLOATS = PART_ROWS * (D + 2);   // one partial: output, maxima, sums
};

enum AttnSite : int {
  SITE_ATTN_Q = 31, SITE_ATTN_Q_EMPTY, SITE_ATTN_KV_FULL, SITE_ATTN_KV_EMPTY, SITE_ATTN_S, SITE_ATTN_P, SITE_ATTN_PV,
  SITE_ATTN_DRAIN, SITE_ATTN_ALIGN, SITE_ATTN_TURN
};

// ------------------------------------------------------------ tcgen05 forms
// K-major B tiles use make_sw128_desc.  v is the B operand of the second
// product with its rows (keys) along K: MN-major, 64 head elements (128 bytes)
// per row, eight-row groups 1024 bytes apart along K (stride byte offset), the
// next 64 elements of the head `lead` bytes away (leading byte offset).
SVD_DEV uint64_t make_sw128_mn_desc(uint32_t saddr, uint32_t lead) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(lead >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

constexpr uint32_t kIdescBMnMajor = 1u << 16;

// The products of one step, issued by one elected lane of a converged warp.
// Descriptors and addresses are the same in every lane, so that the compiler
// can keep them in uniform registers: issued from a branch that one lane takes,
// each MMA cost some 100 cycles of issue, more than it runs for.
// S[128 x N] = Q[128 x 16 K] K^T, both K-major; the next 64 elements of the head
// are 16384 (q) and HALF (k) bytes further on.
template <int K, int HALF>
SVD_DEV void umma_scores(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc) {
#pragma unroll
  for (int k = 0; k < K; ++k)
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc + ((k / 4) * 16384 + (k % 4) * 32) / 16), "l"(b_desc + ((k / 4) * HALF + (k % 4) * 32) / 16),
        "r"(idesc), "r"(k > 0 ? 1 : 0)
        : "memory");
}

// O[128 x N] (+)= P[128 x 64] V[64 x N], P in TMEM (two 16-bit elements per column).
SVD_DEV void umma_values(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem + k * 8), "l"(b_desc + k * 2048 / 16), "r"(idesc), "r"(k > 0 ? 1u : accumulate)
        : "memory");
}

SVD_DEV void umma_commit_elected(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar))
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

// Two fp32 operations in one instruction.
SVD_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

SVD_DEV float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// --------------------------------------------------------------- the cutting
SVD_DEV long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

// sum over i < n of floor((a i + b) / m), a, b >= 0 (the Euclid-like floor sum;
// M: the first modulus, a power of two).
template <int M>
SVD_DEV long long floor_sum(long long n, unsigned a, unsigned b) {
  long long ans = n * (n - 1) / 2 * (a / M) + n * (b / M);
  a %= M;
  b %= M;
  long long y = a * n + b;
  unsigned m = M;
  while (y >= m) {
    n = quotient(y, m);
    b = static_cast<unsigned>(y - n * m);
    const unsigned t = m;
    m = a;
    a = t;
    ans += n * (n - 1) / 2 * (a / m) + n * (b / m);
    a %= m;
    b %= m;
    y = a * n + b;
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

// keys that the first t tokens of the request can see
SVD_DEV int keys_of(const AttnParams& p, const AttnSeq& s, int t) { return p.causal ? min(s.m, max(s.first + t, 0)) : s.m; }
template <int STEP>
SVD_DEV int steps_of(int keys) { return (keys + STEP - 1) / STEP; }
SVD_DEV int tiles_of(const AttnSeq& s, int w) { return (s.n + w - 1) / w; }
// Steps of token tile i of w tokens: at least one, so that rows which see no key are written too.
template <int STEP>
SVD_DEV int tile_steps(const AttnParams& p, const AttnSeq& s, int w, int i) {
  return max(1, steps_of<STEP>(keys_of(p, s, min((i + 1) * w, s.n))));
}
// Steps of the tiles before tile i (i <= tiles).
template <int STEP>
SVD_DEV long long steps_before(const AttnParams& p, const AttnSeq& s, int w, int i) {
  if (!p.causal) return static_cast<long long>(i) * max(1, steps_of<STEP>(s.m));
  long long sum = 0;
  if (i > 0 && i * w >= s.n) {  // the last tile may be cut short
    sum = tile_steps<STEP>(p, s, w, i - 1);
    --i;
  }
  // tiles whose keys fit one step, then ceil((first + (k + 1) w) / step)
  const int room = STEP - s.first;
  const int ones = min(i, room >= w ? room / w : 0);
  sum += ones;
  if (i > ones)
    sum += floor_sum<STEP>(i - ones, static_cast<unsigned>(w),
                           static_cast<unsigned>(s.first + (ones + 1) * w + STEP - 1));
  return sum;
}

// On the line a unit is kUnitCost and its steps long: beginning and ending a
// unit (q, the output) costs about as much as so many steps, and the early
// tiles of a causal prompt are many units of few steps (measured: without it
// the CTAs that got those finished 100 us after the others at 8192 tokens; 3, 4
// and 6 for pairs: chunks behind 5600 keys 64, 65, 69 us, 2 prompts of 2000 tokens
// 110, 103, 103; 1, 2 and 3 for the others: 64-request decoding 91, 84, 86 us).
template <bool PAIR>
constexpr int kUnitCost = PAIR ? 4 : 2;

// A place on the line, and the unit and step it lies in.
struct AttnCut {
  long long at;
  int b, h, tile, j;
  AttnSeq s;
};

// The segment of a unit that a worker is at, and where it goes next.
template <bool PAIR>
struct AttnWalk {
  AttnSeq s;
  int b, h, tile, tiles, j0, j1, steps;
  long long at, end;   // the segment's place on the line; end of this worker's piece

  static constexpr int STEP = PAIR ? 128 : 64;
  SVD_DEV static int tokens(const AttnParams& p) { return PAIR ? 2 * p.tt : p.tt; }
  SVD_DEV bool start(const AttnParams& p, const AttnCut& from, long long to) {
    at = from.at;
    end = to;
    if (at >= end) return false;
    b = from.b;
    h = from.h;
    tile = from.tile;
    j0 = from.j;
    s = from.s;
    tiles = tiles_of(s, tokens(p));
    return open(p);
  }
  SVD_DEV bool open(const AttnParams& p) {
    steps = tile_steps<STEP>(p, s, tokens(p), tile);
    const long long left = end - at - (j0 == 0 ? kUnitCost<PAIR> : 0);
    j1 = left < steps - j0 ? j0 + static_cast<int>(left) : steps;
    return true;
  }
  SVD_DEV bool next(const AttnParams& p) {
    at += j1 - j0 + (j0 == 0 ? kUnitCost<PAIR> : 0);
    if (at >= end) return false;
    j0 = 0;
    if (++tile == tiles) {
      tile = 0;
      if (++h == p.head_groups) {
        h = 0;
        do {
          if (++b >= p.batch) return false;
          s = load_seq(p, b);
        } while (s.n == 0);
        tiles = tiles_of(s, tokens(p));
      }
    }
    return open(p);
  }
  // row tile i: its first token, tokens, steps
  SVD_DEV int t0(const AttnParams& p, int i) const { return tile * tokens(p) + (PAIR ? i * p.tt : 0); }
  SVD_DEV int row_tokens(const AttnParams& p, int i) const { return max(0, min(p.tt, s.n - t0(p, i))); }
  SVD_DEV int row_steps(const AttnParams& p, int i) const {
    const int nt = row_tokens(p, i);
    return nt == 0 ? 0 : steps_of<STEP>(keys_of(p, s, t0(p, i) + nt));
  }
};

// ------------------------------------------------------- the row-wise path
// The tiled product multiplies every value in a tile, and 0 * inf in a masked
// place is a NaN in rows that do not see it.  A row whose sum is finite and whose
// output is not is looked at again: attn_spoilt tells whether a key that it does
// not see, among those of its masked steps, holds such a value, and only then
// attn_row computes it over, without the keys that it does not see.  A value
// that a row rightly sees costs the look alone (a NaN or infinity among its
// scores not even that: its sum is NaN): one prompt of 8192 tokens whose first
// value is NaN 620 us instead of 475.  Rows that are done over take 150 ns a key
// with all eight warps at it (the same prompt with its last value NaN: 77 ms);
// waits elsewhere in the CTA count from the last such row (WaitCtx::progress).

// Whether a row of the request sees key j < m; bits: its mask.
SVD_DEV bool attn_sees(const AttnParams& p, const AttnSeq& s, int token, unsigned long long bits, int j) {
  if (!p.tree) return !p.causal || j <= s.first + token;
  const int node = j - s.first;
  return node < 0 || (p.mask != nullptr ? node < 64 && (bits >> node & 1) != 0 : node <= token);
}

// Where key j lies in k and v, in elements; false where its block is not in the cache.
SVD_DEV bool attn_place(const AttnParams& p, const AttnSeq& s, int b, int kv_head, int j, int d, long long* k_at, long long* v_at) {
  if (p.lens != nullptr) {
    const int page = p.table[b * p.ld_table + (j >> p.block_shift)];
    if (page < 0 || page >= p.num_blocks) return false;
    const long long in = (kv_head * static_cast<long long>(p.block_size) + (j & (p.block_size - 1))) * d;
    *k_at = page * p.k_token + in;
    *v_at = page * p.v_token + in;
  } else {
    *k_at = (s.k0 + j) * p.k_token + kv_head * p.k_head;
    *v_at = (s.k0 + j) * p.v_token + kv_head * p.v_head;
  }
  return true;
}

// Whether a key of [j_lo, j_hi) that this lane's row does not see has a value
// that is not finite.  Called by whole warps of a tile that begins at token t0: a
// lane reads a key, then each asks for its own row.
template <typename T, int D>
__device__ __forceinline__ bool attn_spoilt(const AttnParams& p, const AttnSeq& s, int b, int t0, int token, bool row_ok,
                                         int kv_head, int j_lo, int j_hi) {
  const int lane = static_cast<int>(lane_id());
  const unsigned long long bits = p.mask != nullptr && row_ok ? p.mask[s.q0 + token] : 0;
  j_lo = max(j_lo, p.tree ? s.first : p.causal ? s.first + t0 + 1 : s.m);  // every row of the tile sees the keys before
  bool spoilt = false;
  for (int j0 = j_lo; j0 < j_hi; j0 += 32) {
    float probe = 0.f;  // NaN when any element is not finite
    long long k_at = 0, v_at = 0;
    if (j0 + lane < j_hi && attn_place(p, s, b, kv_head, j0 + lane, D, &k_at, &v_at)) {
      const uint4* v = reinterpret_cast<const uint4*>(static_cast<const T*>(p.v) + v_at);
#pragma unroll 8
      for (int x = 0; x < D / 8; ++x) {
        const uint4 w = v[x];
        const float2 e[4] = {unpack_pair<T>(w.x), unpack_pair<T>(w.y), unpack_pair<T>(w.z), unpack_pair<T>(w.w)};
#pragma unroll
        for (int y = 0; y < 4; ++y) probe = fmaf(e[y].x, 0.f, fmaf(e[y].y, 0.f, probe));
      }
    }
    for (unsigned bad = __ballot_sync(0xffffffffu, probe != 0.f); bad != 0; bad &= bad - 1)
      spoilt = spoilt || !attn_sees(p, s, token, bits, j0 + __ffs(bad) - 1);
  }
  return spoilt;
}

// The output of one row over the keys of [j_lo, j_hi) that it sees, a warp per
// row, 32 keys at a time: a lane takes a key's product with q, then every lane
// its elements of all 32 values.  `base` is the row's maximum, in the exponent's
// units.
template <typename T, int D>
__device__ __forceinline__ void attn_row(const AttnParams& p, const AttnSeq& s, int b, int token, int head, int kv_head,
                                      int j_lo, int j_hi, float base, float (&out)[D / 32]) {
  constexpr int E = D / 32;
  const int lane = static_cast<int>(lane_id());
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (s.q0 + token) * p.q_token + head * p.q_head);
  float o[E] = {};  // not `out`: loads would wait for the stores to it
  const unsigned long long bits = p.mask != nullptr ? p.mask[s.q0 + token] : 0;
  const float c = p.neg ? -p.c : p.c;
  for (int j0 = j_lo; j0 < j_hi; j0 += 32) {
    const int j = j0 + lane;
    long long k_at = 0, v_at = 0;
    const bool seen = j < j_hi && attn_sees(p, s, token, bits, j) && attn_place(p, s, b, kv_head, j, D, &k_at, &v_at);
    float w = 0.f;
    if (seen) {
      const uint4* k = reinterpret_cast<const uint4*>(static_cast<const T*>(p.k) + k_at);
      float2 dot = make_float2(0.f, 0.f);
#pragma unroll 8
      for (int x = 0; x < D / 8; ++x) {
        const uint4 a = q[x], y = k[x];
        dot = fma2(unpack_pair<T>(a.x), unpack_pair<T>(y.x), dot);
        dot = fma2(unpack_pair<T>(a.y), unpack_pair<T>(y.y), dot);
        dot = fma2(unpack_pair<T>(a.z), unpack_pair<T>(y.z), dot);
        dot = fma2(unpack_pair<T>(a.w), unpack_pair<T>(y.w), dot);
      }
      w = exp2f((dot.x + dot.y) * c - base);
    }
    const unsigned all = __ballot_sync(0xffffffffu, seen);
    if (all == 0) continue;
    // keys left out are read at another's place: no branch, so that the loads are in flight together
    const long long other = __shfl_sync(0xffffffffu, v_at, __ffs(all) - 1);
    if (!seen) v_at = other;
#pragma unroll 16
    for (int x = 0; x < 32; ++x) {
      const float weight = __shfl_sync(0xffffffffu, w, x);
      const T* v = static_cast<const T*>(p.v) + __shfl_sync(0xffffffffu, v_at, x) + lane * E;
      const bool one = (all >> x & 1) != 0;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 f = unpack_pair<T>(*reinterpret_cast<const uint32_t*>(v + e));
        o[e] = one ? fmaf(weight, f.x, o[e]) : o[e];
        o[e + 1] = one ? fmaf(weight, f.y, o[e + 1]) : o[e + 1];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = o[e];
}

// The rows of a warp whose output is not finite, over again where a masked place
// has reached them: written where the tiled result was, to the output (whole) or
// to the worker's partial.  Every lane calls it with its own row.
template <typename T, int D, bool PAIR>
__device__ __noinline__ void attn_again(const AttnParams& p, const AttnSeq s, int b, int t0, int token, int head, int kv_head,
                                        int row, bool odd, int j_lo, int j_hi, float base, float inv, float* part,
                                        volatile unsigned long long* progress) {
  constexpr int PART_ROWS = AttnCfg<D, PAIR>::PART_ROWS;
  const int lane = static_cast<int>(lane_id());
  unsigned redo = __ballot_sync(0xffffffffu, attn_spoilt<T, D>(p, s, b, t0, token, odd, kv_head, j_lo, j_hi) && odd);
  while (redo != 0) {
    const int src = __ffs(redo) - 1;
    redo &= redo - 1;
    const int tk = __shfl_sync(0xffffffffu, token, src), hd = __shfl_sync(0xffffffffu, head, src);
    const int rw = __shfl_sync(0xffffffffu, row, src);
    const float bs = __shfl_sync(0xffffffffu, base, src), iv = __shfl_sync(0xffffffffu, inv, src);
    float o[D / 32];
    attn_row<T, D>(p, s, b, tk, hd, kv_head, j_lo, j_hi, bs, o);
    __syncwarp();
#pragma unroll
    for (int e = 0; e < D / 32; ++e) {
      const int d = lane * (D / 32) + e;
      if (part == nullptr)
        static_cast<T*>(p.out)[static_cast<long long>(s.q0 + tk) * p.out_token + hd * p.out_head + d] =
            elem_from_float<T>(o[e] * iv);
      else
        __stcg(part + (PAIR ? (d / 4 * PART_ROWS + rw) * 4 + d % 4 : rw * D + d), o[e]);
    }
    if (lane == 0) *progress = global_timer_ns();
  }
}

// -------------------------------------------------------------- the kernel
struct AttnShared {
  uint64_t q_full[2], q_empty[2], drain[2], turn[2];
  uint64_t s_full[2][2], p_ready[2][2], pv_done[2][2];  // per group and score tile
  uint64_t kv_full[16], kv_empty[16];
  uint32_t slot_info[16];                // what the TMA warp says of a slot's tile
  uint32_t score_info[2][2];             // ... and the MMA warp hands on with the scores
  uint32_t tmem;
  int abort_flag;
  unsigned long long progress;           // when a row was last done over
  AttnCut cut[3];
  long long per;
  long long scan[12];
  long long rem[3];
};

// Bits of a slot's info word.
constexpr uint32_t kInfoRow0 = 1, kInfoRow1 = 2;  // row tiles that the step counts for
constexpr uint32_t kInfoFirst = 4, kInfoLast = 8; // first, last step of the segment
constexpr uint32_t kInfoEnd = 16;                 // k: the worker's last step
constexpr uint32_t kInfoTile = 32;                // always set
constexpr int kInfoValid = 8;                     // v: keys that exist, 0 to 64 (8 bits)
constexpr int kInfoBad = 16;                      // k: blocks of the step outside the cache (16 bits)

// mbar_wait by a whole warp: every lane gets the same answer, so that no lane
// is left alone at a warp-wide instruction.
SVD_DEV bool warp_wait(uint64_t* bar, uint32_t parity, const WaitCtx& ctx, int site, bool honour_abort = true) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, ctx, site, honour_abort));
}

// Every CTA finds its own cuts of the line of steps, one per warpgroup: the
// first steps of its workers and the end of the last one's piece.
template <int WORKERS, bool PAIR>
SVD_DEV void find_cuts(const AttnParams& p, AttnShared* sh) {
  const int k = threadIdx.x >> 7, tid = threadIdx.x & 127;
  const int lane = tid & 31, warp = tid >> 5;
  if (k > WORKERS) return;
  constexpr int STEP = AttnWalk<PAIR>::STEP;
  const int w = AttnWalk<PAIR>::tokens(p);
  long long* scan = sh->scan + k * 4;
  const int rounds = p.batch <= 128 ? 1 : 2;  // more requests than threads: first the total, then the place
  long long total = 0, at = -1;
  for (int round = 0; round < rounds; ++round) {
    long long base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 128) {
      const int b = b0 + tid;
      long long mine = 0;
      long long unit = 0;
      AttnSeq s{};
      if (b < p.batch) {
        s = load_seq(p, b);
        if (s.n > 0) {
          const int tiles = tiles_of(s, w);
          unit = steps_before<STEP>(p, s, w, tiles) + static_cast<long long>(tiles) * kUnitCost<PAIR>;
          mine = unit * p.head_groups;
        }
      }
      long long inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      if (lane == 31) scan[warp] = inc;
      named_barrier_sync(1 + k, 128);
      long long before = base, all = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (x < warp) before += scan[x];
        all += scan[x];
      }
      before += inc - mine;
      base += all;
      if (b0 + 128 < p.batch || round + 1 < rounds) named_barrier_sync(1 + k, 128);
      if (round + 1 == rounds) {
        if (rounds == 1) total = base;
        if (at < 0) {
          const long long workers = static_cast<long long>(gridDim.x) * WORKERS;
          const long long per = max(1ll, quotient(total + workers - 1, workers));
          at = min(per * (static_cast<long long>(blockIdx.x) * WORKERS + k), total);
          if (tid == 0) {
            if (k == 0) sh->per = per;
            sh->cut[k].at = at;
          }
        }
        if (at >= before && at < before + mine) {
          const long long in = at - before;
          const long long h = quotient(in, unit);
          sh->cut[k].s = s;
          sh->cut[k].b = b;
          sh->cut[k].h = static_cast<int>(h);
          sh->rem[k] = in - h * unit;
        }
      }
    }
    total = base;
  }
  named_barrier_sync(1 + k, 128);
  if (warp == 0 && at < total) {
    // the last tile with at most `rem` before it, 32 candidates at a time
    const long long rem = sh->rem[k];
    const AttnSeq s = sh->cut[k].s;
    int lo = 0, hi = tiles_of(s, w);  // lo is at or before it, hi beyond
    if (!p.causal) {
      lo = static_cast<int>(quotient(rem, max(1, steps_of<STEP>(s.m)) + kUnitCost<PAIR>));
    } else {
      while (hi - lo > 1) {
        const int stride = (hi - lo + 31) / 32;
        const int x = lo + lane * stride;
        const bool below = x < hi && steps_before<STEP>(p, s, w, x) + static_cast<long long>(x) * kUnitCost<PAIR> <= rem;
        const int n = __popc(__ballot_sync(0xffffffffu, below));  // lane 0 always
        hi = min(hi, lo + n * stride);
        lo += (n - 1) * stride;
      }
    }
    if (lane == 0) {
      const int in = static_cast<int>(rem - steps_before<STEP>(p, s, w, lo) - static_cast<long long>(lo) * kUnitCost<PAIR>);
      const int steps = tile_steps<STEP>(p, s, w, lo);
      int j = cut_step(in, steps, kUnitCost<PAIR>, p.snap);
      if (j == 0 || j == steps) {  // at the unit's start, or the next one's
        at -= in;
        if (j == steps) {
          j = 0;
          at += steps + kUnitCost<PAIR>;
          if (++lo == tiles_of(s, w)) {
            lo = 0;
            if (++sh->cut[k].h == p.head_groups) {
              sh->cut[k].h = 0;
              int b = sh->cut[k].b;
              AttnSeq behind = s;
              while (++b < p.batch && (behind = load_seq(p, b)).n == 0) {
              }
              sh->cut[k].b = b;  // none where the line ends
              sh->cut[k].s = behind;
            }
          }
        }
        sh->cut[k].at = at;
      }
      sh->cut[k].tile = lo;
      sh->cut[k].j = j;
    }
  }
}

// Joins the partials of divided units: block column c for the unit that worker c
// begins (most begin none), block rows over its rows.  Statistics and outputs of
// several partials are in flight at a time and joined as they come, with a
// running maximum, in the order of the keys.  Latency-bound: 5 us for 8 units of
// 37 partials (8 key/value heads, one token on 65537 keys).  Three CTAs an SM, as
// most have nothing to join (two: 24 ragged prompts 31.1 instead of 30.2 us).
constexpr int kJoinThreads = 256;

template <typename T, int D, bool PAIR>
__global__ void __launch_bounds__(kJoinThreads, 3) attention_join_kernel(const __grid_constant__ AttnParams p) {
  using Cfg = AttnCfg<D, PAIR>;
  grid_dependency_wait();
  const int c0 = blockIdx.x;
  const AttnSplit u = p.splits[c0];
  if (u.more <= 0) return;
  const int warp = threadIdx.x >> 5, lane = static_cast<int>(lane_id());
  const auto partial = [&](int c) -> const float* {
    return p.partials + (2LL * (c0 + c) + (c == 0 ? 1 : 0)) * Cfg::PART_FLOATS;
  };
  const auto row_at = [&](int row) -> T* {  // the output row
    const int r = row & 127;
    return static_cast<T*>(p.out) + static_cast<long long>(u.token0 + (row >> 7) * p.tt + r / p.gp) * p.out_token +
           (u.head0 + r % p.gp) * p.out_head;
  };
  if constexpr (PAIR) {
    // partials [element / 4][row][4]: a lane per row, D / 8 elements per warp
    constexpr int N = D / 32, C = 4;
    for (int row = blockIdx.y * 32 + lane; row < 256; row += gridDim.y * 32) {
      if (row < 128 ? row >= u.rows0 : row - 128 >= u.rows - u.rows0) continue;
      float4 acc[N];
#pragma unroll
      for (int n = 0; n < N; ++n) acc[n] = make_float4(0.f, 0.f, 0.f, 0.f);
      float mm = -INFINITY, ll = 0.f;
#pragma unroll 1
      for (int b0 = 0; b0 <= u.more; b0 += C) {
        float f[C], g[C];
        float4 o[C][N];
#pragma unroll
        for (int k = 0; k < C; ++k) {
          const float* from = partial(min(b0 + k, u.more));
          f[k] = __ldcg(from + Cfg::PART_ROWS * D + row);
          g[k] = __ldcg(from + Cfg::PART_ROWS * (D + 1) + row);
#pragma unroll
          for (int n = 0; n < N; ++n)
            o[k][n] = __ldcg(reinterpret_cast<const float4*>(from) + (warp * N + n) * Cfg::PART_ROWS + row);
        }
        float top = mm;
#pragma unroll
        for (int k = 0; k < C; ++k) top = fmaxf(top, f[k]);  // the last one again where there are fewer
        const float safe = top == -INFINITY ? 0.f : top;
        const float old = exp2_approx(mm - safe);
        mm = top;
        ll *= old;
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n] = make_float4(acc[n].x * old, acc[n].y * old, acc[n].z * old, acc[n].w * old);
#pragma unroll
        for (int k = 0; k < C; ++k) {
          // nothing of what lies behind the last one: by a weight of 0 an infinity would turn into NaN
          const bool one = b0 + k <= u.more;
          const float e = one ? exp2_approx(f[k] - safe) : 0.f;
          ll = fmaf(e, one ? g[k] : 0.f, ll);
#pragma unroll
          for (int n = 0; n < N; ++n) {
            acc[n].x = fmaf(e, one ? o[k][n].x : 0.f, acc[n].x);
            acc[n].y = fmaf(e, one ? o[k][n].y : 0.f, acc[n].y);
            acc[n].z = fmaf(e, one ? o[k][n].z : 0.f, acc[n].z);
            acc[n].w = fmaf(e, one ? o[k][n].w : 0.f, acc[n].w);
          }
        }
      }
      const float iv = ll == 0.f ? 0.f : 1.f / ll;
      uint4* to = reinterpret_cast<uint4*>(row_at(row) + warp * N * 4);
#pragma unroll
      for (int n = 0; n < N; n += 2)
        to[n / 2] = make_uint4(pack_pair<T>(acc[n].x * iv, acc[n].y * iv), pack_pair<T>(acc[n].z * iv, acc[n].w * iv),
                               pack_pair<T>(acc[n + 1].x * iv, acc[n + 1].y * iv),
                               pack_pair<T>(acc[n + 1].z * iv, acc[n + 1].w * iv));
    }
  } else {
    // partials [row][element]: a warp per row, two at head_dim 64
    constexpr int LANES = D / 4, PER = 32 / LANES, C = 16;
    const int sub = lane / LANES, d4 = lane % LANES;
    constexpr int ROWS = kJoinThreads / 32 * PER;
    for (int row = (blockIdx.y * (kJoinThreads / 32) + warp) * PER + sub; row < u.rows; row += gridDim.y * ROWS) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float mm = -INFINITY, ll = 0.f;
#pragma unroll 1
      for (int b0 = 0; b0 <= u.more; b0 += C) {
        float4 o[C];
        float f[C], g[C];
#pragma unroll
        for (int k = 0; k < C; ++k) {
          const float* from = partial(min(b0 + k, u.more));
          f[k] = __ldcg(from + Cfg::PART_ROWS * D + row);
          g[k] = __ldcg(from + Cfg::PART_ROWS * (D + 1) + row);
          o[k] = __ldcg(reinterpret_cast<const float4*>(from + row * D) + d4);
        }
        float top = mm;
#pragma unroll
        for (int k = 0; k < C; ++k) top = fmaxf(top, f[k]);  // the last one again where there are fewer
        const float safe = top == -INFINITY ? 0.f : top;
        const float old = exp2_approx(mm - safe);
        mm = top;
        ll *= old;
        acc = make_float4(acc.x * old, acc.y * old, acc.z * old, acc.w * old);
#pragma unroll
        for (int k = 0; k < C; ++k) {
          const bool one = b0 + k <= u.more;
          const float e = one ? exp2_approx(f[k] - safe) : 0.f;
          ll = fmaf(e, one ? g[k] : 0.f, ll);
          acc.x = fmaf(e, one ? o[k].x : 0.f, acc.x);
          acc.y = fmaf(e, one ? o[k].y : 0.f, acc.y);
          acc.z = fmaf(e, one ? o[k].z : 0.f, acc.z);
          acc.w = fmaf(e, one ? o[k].w : 0.f, acc.w);
        }
      }
      const float iv = ll == 0.f ? 0.f : 1.f / ll;
      *reinterpret_cast<uint2*>(row_at(row) + d4 * 4) =
          make_uint2(pack_pair<T>(acc.x * iv, acc.y * iv), pack_pair<T>(acc.z * iv, acc.w * iv));
    }
  }
}

template <typename T, int D, bool PAGED, bool PAIR>
__global__ void __launch_bounds__(kAttnThreads, 1)
    attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p) {
  using Cfg = AttnCfg<D, PAIR>;
  using Walk = AttnWalk<PAIR>;
  constexpr bool F16 = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t smem[];
  AttnShared* sh = reinterpret_cast<AttnShared*>(smem + Cfg::OFF_BAR);
  static_assert(Cfg::OFF_BAR + sizeof(AttnShared) <= Cfg::SMEM_BYTES && Cfg::SMEM_BYTES <= 232448, "shared memory");
  static_assert(Cfg::WORKERS * Cfg::SLOTS <= 16, "barriers");
  if ((smem_addr(smem) & 1023u) != 0) {  // the swizzle counts from 1024-byte boundaries
    grid_dependency_wait();
    if (threadIdx.x == 0) atomicCAS(p.err, 0, SITE_ATTN_ALIGN);
    if (threadIdx.x < Cfg::WORKERS) p.splits[blockIdx.x * Cfg::WORKERS + threadIdx.x] = AttnSplit{};  // nothing to join
    return;
  }
  const int warp = threadIdx.x >> 5;
  const int lane = static_cast<int>(lane_id());

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh->q_full[i], 1);
      mbar_init(&sh->q_empty[i], Cfg::USERS);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&sh->s_full[i][b], PAGED ? 2 : 1);  // the scores, and what is said of them
        mbar_init(&sh->p_ready[i][b], 128);
        mbar_init(&sh->pv_done[i][b], 1);
      }
      mbar_init(&sh->drain[i], 1);
      mbar_init(&sh->turn[i], 1);
    }
    for (int i = 0; i < Cfg::WORKERS * Cfg::SLOTS; ++i) {
      mbar_init(&sh->kv_full[i], 1);
      mbar_init(&sh->kv_empty[i], Cfg::USERS);
    }
    sh->abort_flag = 0;
    sh->progress = 0;
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
  grid_dependency_wait();
  grid_launch_dependents();
  find_cuts<Cfg::WORKERS, PAIR>(p, sh);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;
  const WaitCtx ctx{&sh->abort_flag, p.err, p.timeout_ns, &sh->progress};
  // softmax group, MMA warp (8, 10) and TMA warp (9, 11) of worker wk
  const int wk = PAIR ? 0 : warp >= 8 ? (warp - 8) >> 1 : warp >> 2;
  Walk w;
  bool more = w.start(p, sh->cut[wk], sh->cut[wk + 1].at);
  constexpr int STEP = Cfg::STEP, AHEAD = Cfg::TILES;  // the scores run AHEAD steps before the values

  if (warp >= 8) {
    if constexpr (PAIR) reg_dealloc<Cfg::OTHER_REGS>();
    uint8_t* ring = smem + Cfg::OFF_KV + wk * Cfg::SLOTS * Cfg::SLOT_BYTES;
    uint64_t* kv_full = sh->kv_full + wk * Cfg::SLOTS;
    uint64_t* kv_empty = sh->kv_empty + wk * Cfg::SLOTS;
    int slot = 0;
    if ((warp & 1) != 0 && (!PAIR || warp == 9)) {
      // ------------------------------------------------------------ TMA warp
      uint32_t phase = 1;  // parity of the next kv_empty wait: the first round finds every slot free
      int ld = 0, seg = 0;
      bool ok = true;
      const auto load = [&](const CUtensorMap* map, const Walk& at, int j, uint32_t info) {
        const int kv_head = at.h * p.gp / p.group, key0 = j * STEP;
        if (!(ok = warp_wait(&kv_empty[slot], phase, ctx, SITE_ATTN_KV_EMPTY))) return;
        uint8_t* dst = ring + slot * Cfg::SLOT_BYTES;
        int page = 0, key = 0;
        const int rows = PAGED ? min(p.block_size, STEP) : STEP;
        if constexpr (PAGED) {
          // a lane per block; a block the table does not name is read out of range, as zeros
          key = key0 + lane * rows;
          page = -1;
          const bool there = lane * rows < STEP && key < at.s.m;
          if (there) page = p.table[at.b * p.ld_table + (key >> p.block_shift)];
          const bool bad = page < 0 || page >= p.num_blocks;
          if (bad) page = p.num_blocks;
          info |= __ballot_sync(0xffffffffu, there && bad) << kInfoBad;
        }
        if (lane == 0) {
          sh->slot_info[wk * Cfg::SLOTS + slot] = info;
          mbar_arrive_expect_tx(&kv_full[slot], Cfg::SLOT_BYTES);
        }
        __syncwarp();
        if constexpr (PAGED) {
          if (lane * rows < STEP)
            for (int hf = 0; hf < Cfg::HALVES; ++hf)
              tma_load_4d_at(map, &kv_full[slot], dst + hf * Cfg::HALF_BYTES + lane * rows * 128, hf * 64,
                             key & (p.block_size - 1), kv_head, page);
        } else {
          if (lane == 0)
            for (int hf = 0; hf < Cfg::HALVES; ++hf)
              tma_load_3d(map, &kv_full[slot], dst + hf * Cfg::HALF_BYTES, hf * 64, kv_head, at.s.k0 + key0);
        }
        ++ld;
        if (++slot == Cfg::SLOTS) {
          slot = 0;
          phase ^= 1;
        }
      };
      // row tiles that step j counts for, and whether it begins or ends the segment
      const auto about = [&](const Walk& at, int j, int st0, int st1) {
        return kInfoTile | (j < st0 ? kInfoRow0 : 0u) | (PAIR && j < st1 ? kInfoRow1 : 0u) | (j == at.j0 ? kInfoFirst : 0u) |
               (j + 1 == at.j1 ? kInfoLast : 0u);
      };
      Walk wv = w;         // v follows k by AHEAD steps
      int jk = w.j0, jv = w.j0;
      int k0 = 0, k1 = 0, v0 = 0, v1 = 0;  // steps of the row tiles
      if (more) {
        k0 = v0 = w.row_steps(p, 0);
        if (PAIR) k1 = v1 = w.row_steps(p, 1);
      }
      bool more_k = more;
      for (int g = 0; more && ok; ++g) {
        if (g >= AHEAD) {
          const int valid = max(0, min(wv.s.m - jv * STEP, STEP));
          load(&map_v, wv, jv, about(wv, jv, v0, v1) | static_cast<uint32_t>(valid) << kInfoValid);
          if (++jv == wv.j1) {
            more = wv.next(p);
            jv = wv.j0;
            v0 = wv.row_steps(p, 0);
            if (PAIR) v1 = wv.row_steps(p, 1);
          }
        }
        if (ok && more_k) {
          if (jk == w.j0) {
            if (!(ok = warp_wait(&sh->q_empty[wk], (seg & 1) ^ 1, ctx, SITE_ATTN_Q_EMPTY))) break;
            if (lane == 0) {
              constexpr int QT = PAIR ? 2 : 1;
              mbar_arrive_expect_tx(&sh->q_full[wk], static_cast<uint32_t>(QT * Cfg::HALVES * p.tt * p.gp * 128));
              for (int i = 0; i < QT; ++i)
                for (int hf = 0; hf < Cfg::HALVES; ++hf)
                  tma_load_4d_at(&map_q, &sh->q_full[wk], smem + (wk + i) * Cfg::Q_BYTES + hf * (128 * 128), hf * 64, 0,
                                 w.h, w.s.q0 + w.t0(p, i));
            }
            ++seg;
          }
          const uint32_t info = about(w, jk, k0, k1);
          Walk now = w;
          const int j = jk;
          if (++jk == w.j1) {
            more_k = w.next(p);
            jk = w.j0;
            k0 = w.row_steps(p, 0);
            if (PAIR) k1 = w.row_steps(p, 1);
          }
          load(&map_k, now, j, info | (more_k ? 0u : kInfoEnd));
        }
      }
      // every load in flight has landed before the CTA ends
      for (int sl = 0; sl < Cfg::SLOTS; ++sl)
        if (ld > sl) {
          const int round = (ld - 1 - sl) / Cfg::SLOTS;
          mbar_wait(&kv_full[sl], static_cast<uint32_t>(round & 1), ctx, SITE_ATTN_DRAIN, false);
        }
      if (seg > 0) mbar_wait(&sh->q_full[wk], static_cast<uint32_t>((seg - 1) & 1), ctx, SITE_ATTN_DRAIN, false);
    } else if ((warp & 1) == 0) {
      // ------------------------------------------------------------ MMA warp
      // One per row tile.  In PAIR the two take turns, P V and then Q K of one
      // tile at a time: the products of a tile run while the other warp waits
      // for its probabilities and its tiles of k and v.  (Issued as they come,
      // the products of the tiles alternate on the tensor pipe, both groups get
      // their scores at the same time and both want the exponential unit at the
      // same time: 2200 cycles for 128 keys instead of 1150.  Issued by one warp
      // for both, its waits came between the products: 70 us for the chunks behind
      // 5600 keys instead of 68.)
      const int i = (warp - 8) >> 1;           // group
      constexpr uint32_t idesc_s = make_idesc_16bit(128, STEP, F16);
      constexpr uint32_t idesc_o = make_idesc_16bit(128, D, F16) | kIdescBMnMajor;
      const uint64_t q_desc = make_sw128_desc(smem_addr(smem + i * Cfg::Q_BYTES));
      const uint64_t k_desc = make_sw128_desc(smem_addr(ring));
      const uint64_t v_desc = make_sw128_mn_desc(smem_addr(ring), Cfg::HALF_BYTES);
      const uint32_t mine = PAIR && i == 1 ? kInfoRow1 : kInfoRow0;
      const uint32_t t_s = tmem + i * 128, t_o = tmem + 256 + i * D;
      const volatile uint32_t* slot_info = sh->slot_info + wk * Cfg::SLOTS;
      uint32_t phase = 0, q_phase = 0, turn = i == 0 ? 1 : 0;
      unsigned n_q = 0, n_p = 0;               // score and probability tiles so far
      bool ok = true, had = false;             // had: P V in this segment (PAIR)
      // waits for the next slot of the ring, in the order of the loads
      const auto take = [&](uint32_t* info) -> int {
        ok = ok && warp_wait(&kv_full[slot], phase, ctx, SITE_ATTN_KV_FULL);
        const int got = slot;
        *info = slot_info[got];
        if (++slot == Cfg::SLOTS) {
          slot = 0;
          phase ^= 1;
        }
        return got;
      };
      const auto wait_p = [&](int hf) {
        // one barrier per 64 probabilities: the halves of a tile, or the two tiles in turn
        const int b = PAIR ? hf : n_p & 1;
        ok = ok && warp_wait(&sh->p_ready[i][b], PAIR ? n_p & 1 : n_p >> 1 & 1, ctx, SITE_ATTN_P);
      };
      const auto take_turn = [&] {
        if constexpr (PAIR) {
          ok = ok && warp_wait(&sh->turn[i], turn, ctx, SITE_ATTN_TURN);
          turn ^= 1;
        }
      };
      const auto pass_turn = [&] {
        if constexpr (PAIR) {
          if (lane == 0) mbar_arrive(&sh->turn[i ^ 1]);
          __syncwarp();
        }
      };
      int stop = more ? INT_MAX : 0;           // known once the last k has come
      for (int g = 0; g < stop; ++g) {         // P V(g - AHEAD) and Q K(g)
        uint32_t iv = 0, ik = 0;
        int sv = 0, sk = 0;
        if (g >= AHEAD) {
          sv = take(&iv);
          const int valid = iv >> kInfoValid & 0xff;
          if (ok && valid < STEP && (!PAIR || i == 0)) {
            // rows behind the last key are other requests' or nobody's: zeros
            uint8_t* t = ring + sv * Cfg::SLOT_BYTES;
            for (int x = valid * 8 + lane; x < STEP * 8; x += 32)
              for (int hf = 0; hf < Cfg::HALVES; ++hf)
                *reinterpret_cast<uint4*>(t + hf * Cfg::HALF_BYTES + x * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        if (stop == INT_MAX) {
          sk = take(&ik);
          if ((ik & kInfoEnd) != 0) stop = g + 1 + AHEAD;
        }
        if ((iv & mine) != 0) wait_p(0);
        take_turn();
        if (!ok) break;
        if ((iv & mine) != 0) {                // O (+)= P V, 64 keys at a time
#pragma unroll
          for (int hf = 0; hf < STEP / 64; ++hf) {
            if (hf > 0) wait_p(hf);
            if (!ok) break;
            tc_fence_after();
            umma_values(t_o, t_s + (PAIR ? hf * 32 : (n_p & 1) * 64),
                        v_desc + (sv * Cfg::SLOT_BYTES + hf * 64 * 128) / 16, idesc_o, hf > 0 || (iv & kInfoFirst) == 0);
          }
          if (!ok) break;
          if (!PAIR) umma_commit_elected(&sh->pv_done[i][n_p & 1]);
          ++n_p;
          had = true;
        }
        if (PAIR && (iv & kInfoLast) != 0) {
          // only for a segment with steps for this tile: their probabilities hold
          // the barrier's next phase back until every row has seen this one
          if (had) umma_commit_elected(&sh->pv_done[i][0]);
          had = false;
        }
        if ((ik & kInfoFirst) != 0) {          // q comes late: the other tile's P V before it
          pass_turn();
          take_turn();
          ok = ok && warp_wait(&sh->q_full[wk], q_phase, ctx, SITE_ATTN_Q);
          q_phase ^= 1;
          if (!ok) break;
        }
        if ((ik & mine) != 0) {                // S = Q K^T
          const int b = PAIR ? 0 : n_q & 1;
          tc_fence_after();
          umma_scores<D / 16, Cfg::HALF_BYTES>(t_s + b * 64, q_desc, k_desc + sk * (Cfg::SLOT_BYTES / 16), idesc_s);
          umma_commit_elected(&sh->s_full[i][b]);
          if (PAGED && lane == 0) {
            sh->score_info[i][b] = ik;
            mbar_arrive(&sh->s_full[i][b]);
          }
          ++n_q;
        }
        pass_turn();
        if (g >= AHEAD) umma_commit_elected(&kv_empty[sv]);
        if (ik != 0) umma_commit_elected(&kv_empty[sk]);
        if ((ik & kInfoLast) != 0) umma_commit_elected(&sh->q_empty[wk]);  // the last product with this q is issued
      }
      umma_commit_elected(&sh->drain[i]);
      __syncwarp();
      mbar_wait(&sh->drain[i], 0, ctx, SITE_ATTN_DRAIN, false);
    }
  } else {
    // -------------------------------------------------------- softmax groups
    if constexpr (PAIR) reg_alloc<Cfg::SOFTMAX_REGS>();
    const int i = warp >> 2;                          // group: row tile, S and O
    const int r = threadIdx.x & 127;                  // row of the tile, lane of TMEM
    const int ti = PAIR ? i : 0;                      // row tile of the unit
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + i * 128, t_o = tmem + lanes + 256 + i * D;
    const int row_token = r / p.gp, row_head = r - row_token * p.gp;
    unsigned n_s = 0, n_seg = 0;                      // score tiles taken, segments with any
    bool ok = true;
    AttnSplit split{};
    for (; more; more = w.next(p)) {
      const int steps_i = w.row_steps(p, ti);
      const int t0 = w.t0(p, ti), token = t0 + row_token;
      const bool row_ok = row_token < w.row_tokens(p, ti);
      const bool warp_ok = __any_sync(0xffffffffu, row_ok);
      // keys below `open` are seen by every row of the tile, keys from `sees` on by none of this row (outside a mask)
      const int open = min(w.s.m, p.tree ? w.s.first : p.causal ? w.s.first + t0 + 1 : w.s.m);
      const int sees = min(w.s.m, p.tree ? (p.mask != nullptr ? w.s.first : w.s.first + token + 1)
                                         : p.causal ? w.s.first + token + 1 : w.s.m);
      const unsigned long long bits = p.mask != nullptr && row_ok ? p.mask[w.s.q0 + token] : 0;
      float m = -INFINITY, l = 0.f;                   // m in units of the scores
      bool some = false;
      const int last_j = min(w.j1, steps_i);
      for (int j = w.j0; j < last_j; ++j) {
        const int sb = PAIR ? 0 : n_s & 1;
        if (!(ok = warp_wait(&sh->s_full[i][sb], (PAIR ? n_s : n_s >> 1) & 1, ctx, SITE_ATTN_S))) break;
        if (!warp_ok) {                               // rows of nobody: their probabilities stay what they are
          mbar_arrive(&sh->p_ready[i][sb]);
          if (PAIR) mbar_arrive(&sh->p_ready[i][1]);
          ++n_s;
          continue;
        }
        tc_fence_after();
        const uint32_t t_sb = t_s + sb * 64;
        float s[STEP];
#pragma unroll
        for (int x = 0; x < STEP; x += 32) tmem_ld_x32(t_sb + x, reinterpret_cast<uint32_t(&)[32]>(s[x]));
        tmem_ld_wait();
        if (p.neg) {
#pragma unroll
          for (int x = 0; x < STEP; ++x) s[x] = -s[x];
        }
        const int rel = j * STEP;
        unsigned bad_pages = 0;
        if constexpr (PAGED) bad_pages = *const_cast<volatile uint32_t*>(&sh->score_info[i][sb]) >> kInfoBad;
        if (rel + STEP > open || bad_pages != 0) {
          // one bit per key of the step
          uint32_t vis[STEP / 32];
#pragma unroll
          for (int x = 0; x < STEP / 32; ++x) {
            const int lim = sees - rel - 32 * x;
            vis[x] = lim >= 32 ? 0xffffffffu : lim > 0 ? (1u << lim) - 1u : 0u;
          }
          if (p.mask != nullptr) {
            // the tree's 64 bits, moved to where its first key lies in this step
            const int at = w.s.first - rel;
#pragma unroll
            for (int x = 0; x < STEP / 32; ++x) {
              const int by = at - 32 * x;             // bit 0 of the tree in this word's coordinates
              uint32_t part = 0;
              if (by > -64 && by < 32) part = by >= 0 ? static_cast<uint32_t>(bits << by) : static_cast<uint32_t>(bits >> -by);
              const int end = w.s.m - rel - 32 * x;   // keys that exist
              part &= end >= 32 ? 0xffffffffu : end > 0 ? (1u << end) - 1u : 0u;
              vis[x] |= part;
            }
          }
          if constexpr (PAGED) {
            const int rows = min(p.block_size, STEP);
            for (unsigned rest = bad_pages; rest != 0; rest &= rest - 1) {
              const int lo = (__ffs(rest) - 1) * rows;
#pragma unroll
              for (int x = 0; x < STEP / 32; ++x) {
                const int a = max(lo - 32 * x, 0), z = min(lo + rows - 32 * x, 32);
                if (a < z) vis[x] &= ~((z - a == 32 ? 0xffffffffu : (1u << (z - a)) - 1u) << a);
              }
            }
          }
#pragma unroll
          for (int x = 0; x < STEP; ++x)
            if (!(vis[x / 32] >> (x % 32) & 1u)) s[x] = -INFINITY;
        }
        float tops[4] = {s[0], s[1], s[2], s[3]};     // independent chains
#pragma unroll
        for (int x = 4; x < STEP; x += 8) {
#pragma unroll
          for (int y = 0; y < 4; ++y)
            tops[y] = x + 4 < STEP ? fmaxf(tops[y], fmaxf(s[x + y], s[x + 4 + y])) : fmaxf(tops[y], s[x + y]);
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        // a new base only where the maximum has grown by more than the stale one absorbs
        const bool grow = top > m && (m == -INFINITY || (top - m) * p.c > kAttnLazy);
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? exp2_approx((m - top) * p.c) : 1.0f;
          if (grow) {
            m = top;
            l *= alpha;
          }
          if (some) {
            if constexpr (!PAIR) {                    // PAIR: the scores came after P V of the step before
              const unsigned last = n_s - 1;
              if (!(ok = warp_wait(&sh->pv_done[i][last & 1], last >> 1 & 1, ctx, SITE_ATTN_PV))) break;
              tc_fence_after();
            }
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
        const float neg_base = m == -INFINITY ? 0.f : -m * p.c;
        float2 part_sums[2] = {};                     // two chains (one 68, two 65 us for the chunks behind 5600 keys)
#pragma unroll
        for (int hf = 0; hf < STEP / 64; ++hf) {
          uint32_t pk[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            float2 e = fma2(make_float2(s[hf * 64 + 2 * x], s[hf * 64 + 2 * x + 1]), make_float2(p.c, p.c),
                            make_float2(neg_base, neg_base));
            e.x = exp2_approx(e.x);
            e.y = exp2_approx(e.y);
            part_sums[x & 1] = add2(part_sums[x & 1], e);
            pk[x] = pack_pair<T>(e.x, e.y);
          }
          tmem_st_x32(t_sb + hf * 32, pk);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&sh->p_ready[i][PAIR ? hf : sb]);
        }
        const float2 sums = add2(part_sums[0], part_sums[1]);
        l += sums.x + sums.y;
        ++n_s;
        some = true;
      }
      ok = __all_sync(0xffffffffu, ok && *ctx.abort_flag == 0);
      if (!ok) break;
      if (PAIR ? last_j > w.j0 : some) {
        const unsigned last = n_s - 1;
        if (!(ok = warp_wait(&sh->pv_done[i][PAIR ? 0 : last & 1], PAIR ? n_seg & 1 : last >> 1 & 1, ctx, SITE_ATTN_PV))) break;
        tc_fence_after();
        ++n_seg;
      }
      // ---------------------------------------------------- the segment's end
      const bool whole = w.j0 == 0 && w.j1 == w.steps;
      const float base = m == -INFINITY ? 0.f : m * p.c;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int row = ti * 128 + r;
      const int head = w.h * p.gp + row_head, kv_head = w.h * p.gp / p.group;
      // partials of this worker: one for the unit that it begins, one for the unit that it goes on with
      float* part = p.partials + ((static_cast<long long>(blockIdx.x) * Cfg::WORKERS + wk) * 2 + (w.j0 == 0 ? 1 : 0)) *
                                     Cfg::PART_FLOATS;
      T* dst = static_cast<T*>(p.out) + static_cast<long long>(w.s.q0 + token) * p.out_token + head * p.out_head;
      if (warp_ok) {
        float probe = 0.f;                            // NaN when any output is not finite
#pragma unroll 1
        for (int x = 0; x < D; x += 32) {
          uint32_t v[32];
          tmem_ld_x32(t_o + x, v);
          tmem_ld_wait();
          if (!some) {
#pragma unroll
            for (int y = 0; y < 32; ++y) v[y] = 0;
          }
#pragma unroll
          for (int y = 0; y < 32; ++y) probe = fmaf(__uint_as_float(v[y]), 0.f, probe);
          if (row_ok) {
            if (whole) {
#pragma unroll
              for (int y = 0; y < 32; y += 16) {
                uint32_t o[8];
#pragma unroll
                for (int z = 0; z < 8; ++z)
                  o[z] = pack_pair<T>(__uint_as_float(v[y + 2 * z]) * inv, __uint_as_float(v[y + 2 * z + 1]) * inv);
                reinterpret_cast<uint4*>(dst + x + y)[0] = make_uint4(o[0], o[1], o[2], o[3]);
                reinterpret_cast<uint4*>(dst + x + y)[1] = make_uint4(o[4], o[5], o[6], o[7]);
              }
            } else {
#pragma unroll
              for (int y = 0; y < 32; y += 8) {
                if constexpr (PAIR) {  // [element / 4][row][4]: many rows, a warp writes whole lines
                  float4* at = reinterpret_cast<float4*>(part) + (x + y) / 4 * Cfg::PART_ROWS + row;
                  __stcg(at, make_float4(__uint_as_float(v[y]), __uint_as_float(v[y + 1]), __uint_as_float(v[y + 2]),
                                         __uint_as_float(v[y + 3])));
                  __stcg(at + Cfg::PART_ROWS, make_float4(__uint_as_float(v[y + 4]), __uint_as_float(v[y + 5]),
                                                          __uint_as_float(v[y + 6]), __uint_as_float(v[y + 7])));
                } else {               // [row][element]: few rows, a warp reads whole rows
                  __stcg(reinterpret_cast<uint4*>(part + row * D + x + y), make_uint4(v[y], v[y + 1], v[y + 2], v[y + 3]));
                  __stcg(reinterpret_cast<uint4*>(part + row * D + x + y) + 1,
                         make_uint4(v[y + 4], v[y + 5], v[y + 6], v[y + 7]));
                }
              }
            }
          }
        }
        if (!whole && row_ok) {
          __stcg(part + Cfg::PART_ROWS * D + row, m == -INFINITY ? -INFINITY : base);
          __stcg(part + Cfg::PART_ROWS * (D + 1) + row, l);
        }
        // rows that a masked place may have reached (a sum that is not finite: rightly so)
        const bool odd = row_ok && probe != 0.f && l == l;
        if (__any_sync(0xffffffffu, odd))
          attn_again<T, D, PAIR>(p, w.s, w.b, t0, token, head, kv_head, row, odd, w.j0 * STEP, min(w.j1 * STEP, w.s.m), base,
                                 inv, whole ? nullptr : part, &sh->progress);
      }
      tc_fence_before();
      if (!whole && w.j0 == 0) {                      // the worker's last segment: others go on with the unit
        const long long unit = w.at + kUnitCost<PAIR>;
        split.more = static_cast<int>(quotient(unit + w.steps - 1, sh->per) - quotient(unit, sh->per));
        split.rows0 = w.row_tokens(p, 0) * p.gp;
        split.rows = split.rows0 + (PAIR ? w.row_tokens(p, 1) * p.gp : 0);
        split.token0 = w.s.q0 + w.t0(p, 0);
        split.head0 = w.h * p.gp;
      }
    }
    if (r == 0 && ti == 0) p.splits[blockIdx.x * Cfg::WORKERS + wk] = ok ? split : AttnSplit{};
  }

  // rows of no request give zeros
  {
    const int lo = min(max(p.cu_q[0], 0), p.q_tokens), hi = min(max(p.cu_q[p.batch], lo), p.q_tokens);
    const int heads = p.head_groups * p.gp;
    const long long rows = static_cast<long long>(lo + p.q_tokens - hi) * heads;
    for (long long x = blockIdx.x * static_cast<long long>(kAttnThreads) + threadIdx.x; x < rows;
         x += static_cast<long long>(gridDim.x) * kAttnThreads) {
      const int t = static_cast<int>(x / heads), h = static_cast<int>(x % heads);
      T* dst = static_cast<T*>(p.out) + static_cast<long long>(t < lo ? t : t - lo + hi) * p.out_token + h * p.out_head;
      for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
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
