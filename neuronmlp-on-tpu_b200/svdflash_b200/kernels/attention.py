"""The attention half of a decoder layer on the B200 kernels.

The reference runs its MLP inside a LLaMA decoder layer (models/modeling_llama.py:
rotary positions, KV cache, grouped-query attention; bench/e2e_block.py:208-229
for the prefill block).  These are its operators here, for serving:

* ``rope_cache`` / ``rope``: rotary positions, with the keys and values written
  into a paged cache in the same pass; ``rope_frequencies`` gives the tables of
  contexts stretched beyond the trained length;
* ``prompt_attention``: causal attention over packed prompts;
* ``tree_attention``: attention of each request's newest tokens (one token, a
  chain, or a tree of drafted tokens) over the paged cache;
* ``page_step``: block tables, slots and positions from request lengths, on the
  GPU; ``tree_positions`` turns its positions into those of drafted trees.

Tensors are CUDA tensors, activations bf16 or fp16 ``[tokens, heads, head_dim]``
with any token and head strides (views of one q|k|v projection are read in
place).  A layer's cache is two tensors ``[num_blocks, kv_heads, block_size,
head_dim]``.  Softmax statistics and sums are fp32.  The work goes to the
current stream of the tensors' device and nothing synchronises, so a step can
be captured in a CUDA graph.  There is no CPU path and no backward (the library
is for inference).
"""
from __future__ import annotations

import math
import threading
from typing import NamedTuple, Optional, Tuple

import torch

from .. import _lib
from . import ops

__all__ = ["PageStep", "kv_cache", "page_step", "prompt_attention", "rope", "rope_cache", "rope_frequencies",
           "tree_attention", "tree_positions"]

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


# -------------------------------------------------------------------- checks
# A call first takes its arguments through one expression of plain attribute
# comparisons (a decoding step's launches take a few microseconds each, so the
# checks have to as well); only where that fails, _refuse_* name what is wrong.
_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice
_thread = threading.get_ident
_capturing = torch._C._cuda_isCurrentStreamCapturing
_PLAIN = torch.contiguous_format
_MASK_BITS = 64  # tree tokens that a row's mask names


def _refuse_dtype(t) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"expected a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"supported dtypes are bfloat16 and float16, got {t.dtype}")


def _refuse_heads(**tensors: torch.Tensor) -> None:
    """Raises what is wrong with [tokens, heads, head_dim] tensors; the first sets the type, device and head size."""
    like = None
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
        if t.dim() != 3 or t.shape[1] <= 0 or t.shape[2] <= 0:
            raise ValueError(f"{name}: expected [tokens, heads, head_dim], got {tuple(t.shape)}")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (the B200 path has no CPU fallback)")
        if like is None:
            _refuse_dtype(t)
            like = t
        if t.dtype != like.dtype:
            raise TypeError("all inputs must have the same dtype")
        if t.device != like.device:
            raise ValueError("inputs must be CUDA tensors on one device")
        if t.shape[2] != like.shape[2]:
            raise ValueError(f"{name} has head_dim {t.shape[2]}, expected {like.shape[2]}: dimensions do not match")


def _vector_rows(t: torch.Tensor, strides) -> bool:
    """Whether the kernels read t's rows in place: unit stride in the head, rows on 16-byte boundaries."""
    return (strides[2] == 1 and not (strides[0] | strides[1]) & 7 and not t.data_ptr() & 15
            and (strides[0] > 0 or t.shape[0] == 1) and (strides[1] > 0 or t.shape[1] == 1))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t`, or a copy of it that the kernels read in place."""
    if _vector_rows(t, t.stride()):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _index(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device) -> torch.Tensor:
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == device.index and t.is_contiguous():
            return t
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype:
        raise TypeError(f"{name} must be a {str(dtype)[6:]} tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}: dimensions do not match")
    if t.device != device:
        raise ValueError("inputs must be CUDA tensors on one device")
    return t if t.is_contiguous() else t.contiguous()


def _offsets(name: str, t: torch.Tensor, device: torch.device) -> torch.Tensor:
    try:
        if (t.dtype is torch.int32 and t.dim() == 1 and t.shape[0] > 1 and t.get_device() == device.index
                and t.is_contiguous()):
            return t
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32:
        raise TypeError(f"{name} must be an int32 tensor")
    if t.dim() != 1 or t.shape[0] < 2:
        raise ValueError(f"{name} must be [batch + 1], got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError("inputs must be CUDA tensors on one device")
    return t if t.is_contiguous() else t.contiguous()


def _refuse_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, like: torch.Tensor, kv_heads: Optional[int]) -> None:
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
        if t.dim() != 4 or min(t.shape) <= 0:
            raise ValueError(f"{name}: expected [num_blocks, kv_heads, block_size, head_dim], got {tuple(t.shape)}")
        if t.dtype != like.dtype:
            raise TypeError("all inputs must have the same dtype")
        if t.device != like.device:
            raise ValueError("inputs must be CUDA tensors on one device")
        if t.shape[3] != like.shape[2] or (kv_heads is not None and t.shape[1] != kv_heads):
            raise ValueError(f"{name} {tuple(t.shape)} does not match the heads: dimensions do not match")
        if t.stride()[1:] != (t.shape[2] * t.shape[3], t.shape[3], 1):
            raise ValueError(f"{name} must be contiguous inside a block")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have matching shapes")


def _check_caches(k_cache, v_cache, like: torch.Tensor, kv_heads: Optional[int]):
    """(num_blocks, kv_heads, block_size, stride between k blocks, between v blocks), or an exception."""
    try:
        nb, hk, bs, d = shape = k_cache.shape
        kb, k1, k2, k3 = k_cache.stride()
        vb, v1, v2, v3 = v_cache.stride()
        if (k3 == v3 == 1 and k2 == v2 == d and k1 == v1 == bs * d and v_cache.shape == shape and nb * hk * bs > 0
                and d == like.shape[2] and (kv_heads is None or hk == kv_heads)
                and k_cache.dtype is v_cache.dtype is like.dtype
                and k_cache.get_device() == v_cache.get_device() == like.get_device()):
            return nb, hk, bs, kb, vb
    except (AttributeError, TypeError, ValueError):
        pass
    _refuse_caches(k_cache, v_cache, like, kv_heads)
    raise ValueError("k_cache and v_cache must have matching layouts")


def _scale(scale: Optional[float], head_dim: int) -> float:
    if scale is None:
        return 1.0 / math.sqrt(head_dim)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    return float(scale)


def _output(out: torch.Tensor, q: torch.Tensor) -> torch.Tensor:
    if out.shape != q.shape or out.device != q.device:
        raise ValueError(f"out must be {tuple(q.shape)} on {q.device}: dimensions do not match")
    if out.dtype != q.dtype:
        raise TypeError("out must have the inputs' dtype")
    if not _vector_rows(out, out.stride()):
        raise ValueError("out must have 16-byte aligned rows")
    return out


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors [tokens, heads, elements] of one type with unit stride in the last dimension share a place."""
    (a_n, a_heads, a_row), (b_n, b_heads, b_row) = a.shape, b.shape
    a_token, b_token = (t.stride(0) if t.shape[0] > 1 else 0 for t in (a, b))
    a_head, b_head = (t.stride(1) if t.shape[1] > 1 else 0 for t in (a, b))
    ahead = (b.data_ptr() - a.data_ptr()) // a.element_size()
    a_heads, b_heads = (a_heads - 1) * a_head + a_row, (b_heads - 1) * b_head + b_row      # places of a token's heads
    a_tokens, b_tokens = (a_n - 1) * a_token + a_row, (b_n - 1) * b_token + b_row          # of a head's tokens
    if a_tokens + a_heads - a_row <= ahead or b_tokens + b_heads - b_row <= -ahead:
        return False
    # views of one buffer that lie side by side or take turns: b at the same place between two rows, between two
    # tokens or between two heads of a
    for period, mine, other in ((math.gcd(a_token, b_token, a_head, b_head), a_row, b_row),
                                (a_token if a_token == b_token else 0, a_heads, b_heads),
                                (a_head if a_head == b_head else 0, a_tokens, b_tokens)):
        if period and mine <= ahead % period <= period - other:
            return False
    # whatever else: the rows of both in the order of their places, each against the ends of the other's before it
    a_at, b_at = ((start + torch.arange(t.shape[0])[:, None] * token + torch.arange(t.shape[1]) * head).flatten()
                  for t, start, token, head in ((a, 0, a_token, a_head), (b, ahead, b_token, b_head)))
    places, order = torch.cat((a_at, b_at)).sort(stable=True)
    of_a = order < a_at.numel()
    before = torch.iinfo(torch.int64).min
    a_end = torch.where(of_a, places + a_row, before).cummax(0).values
    b_end = torch.where(of_a, before, places + b_row).cummax(0).values
    return bool((torch.where(of_a, b_end, a_end) > places).any())


def _apart(out: torch.Tensor, *inputs: torch.Tensor) -> None:
    """Refuses an `out` that shares memory with inputs that the kernels read while they write it."""
    if out.numel() and any(t.numel() and _overlap(out, t) for t in inputs):
        raise ValueError("out must not overlap the inputs")


def _call(fn, args: bytes, device: torch.device, what: str) -> None:
    index = device.index
    if index != _device():
        with torch.cuda.device(device):
            status = fn(args, _stream(index))
    else:
        status = fn(args, _stream(index))
    if status:
        _lib.check(status, what)


_workspace_need: dict = {}


def _workspace(device: torch.device, head_dim: int):
    """The attention workspace of the device's current stream and this thread: the pool that the other operators use."""
    need = _workspace_need.get((device.index, head_dim))
    if need is None:
        lib = _lib.load()
        with torch.cuda.device(device):
            need = max(int(lib.svdmlp_prompt_workspace_bytes()), int(lib.svdmlp_tree_workspace_bytes(head_dim)))
        _workspace_need[device.index, head_dim] = need
    # the usual case without a lock: reading the pool is one step
    index = device.index
    ws = ops._ws_pool.get((index, _stream(index), _thread()))
    if ws is not None and ws.nbytes >= need and index == _device() and not _capturing():
        return ws
    return ops.workspace_for(device, need)


# -------------------------------------------------------------------- rotary
def rope_frequencies(head_dim: int, *, base: float = 10000.0, rotary_dim: Optional[int] = None,
                     scaling: Optional[dict] = None, device="cuda") -> Tuple[torch.Tensor, float]:
    """(inv_freq [rotary_dim / 2] fp32, scale) of rotary positions.

    `scaling` stretches the context, with a checkpoint's own keys
    (``rope_type`` or ``type``):

    * ``linear``: every frequency divided by ``factor``;
    * ``llama3``: frequencies whose wavelength exceeds
      ``original_max_position_embeddings / low_freq_factor`` divided by
      ``factor``, those below ``original / high_freq_factor`` kept, a linear
      blend of the two between;
    * ``yarn``: the same between the pairs that turn ``beta_fast`` (32) and
      ``beta_slow`` (1) times over the original context, linear in the pair's
      index, from whole pairs unless ``truncate`` is false, and a magnitude of
      0.1 ln(factor) + 1; with ``mscale`` and ``mscale_all_dim`` the quotient of
      0.1 mscale ln(factor) + 1 and the same of mscale_all_dim;
      ``attention_factor`` overrides both.
    """
    rot = head_dim if rotary_dim is None else rotary_dim
    if isinstance(rot, bool) or not isinstance(rot, int) or rot <= 0 or rot % 2 or rot > head_dim:
        raise ValueError(f"rotary_dim must be a positive even integer of at most head_dim, got {rot}")
    if not base > 0:
        raise ValueError(f"base must be positive, got {base}")
    half = rot // 2
    freq = [base ** (-i / half) for i in range(half)]
    magnitude = 1.0
    kind = "default" if not scaling else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "linear":
        freq = [f / scaling["factor"] for f in freq]
    elif kind == "llama3":
        factor, context = scaling["factor"], scaling["original_max_position_embeddings"]
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        if high <= low:
            raise ValueError("high_freq_factor must exceed low_freq_factor")
        turns = [f * context / (2 * math.pi) for f in freq]
        keep = [min(1.0, max(0.0, (t - low) / (high - low))) for t in turns]
        freq = [f * (k + (1 - k) / factor) for f, k in zip(freq, keep)]
    elif kind == "yarn":
        factor, context = scaling["factor"], scaling["original_max_position_embeddings"]

        def pair_that_turns(times):
            return half * math.log(context / (2 * math.pi * times)) / math.log(base)

        def magnitude_of(times):
            return 0.1 * times * math.log(factor) + 1.0 if factor > 1 else 1.0

        first, last = pair_that_turns(scaling.get("beta_fast", 32)), pair_that_turns(scaling.get("beta_slow", 1))
        if scaling.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rot - 1)
        span = max(last - first, 0.001)
        keep = [1 - min(1.0, max(0.0, (i - first) / span)) for i in range(half)]
        freq = [f * (k + (1 - k) / factor) for f, k in zip(freq, keep)]
        scales = scaling.get("mscale"), scaling.get("mscale_all_dim")
        if scaling.get("attention_factor"):
            magnitude = scaling["attention_factor"]
        elif all(scales):
            magnitude = magnitude_of(scales[0]) / magnitude_of(scales[1])
        elif scales[0] not in (None, 1) or scales[1] is not None:
            raise ValueError("mscale and mscale_all_dim go together: one of them alone has no one meaning")
        else:
            magnitude = magnitude_of(1.0)
    elif kind != "default":
        raise ValueError(f"unknown rotary scaling {kind!r} (default, linear, llama3, yarn)")
    return torch.tensor(freq, dtype=torch.float32, device=device), float(magnitude)


def _rope(q, k, v, positions, slots, inv_freq, k_cache, v_cache, interleaved, scale, return_k):
    cached = k_cache is not None or v_cache is not None
    try:
        n, h, d = q.shape
        nk, hk, dk = k.shape
        device, dtype = q.device, q.dtype
        code = _DTYPES.get(dtype)
        good = (code is not None and dk == d and h > 0 and hk > 0 and d > 0 and k.dtype is dtype and k.device == device
                and q.is_cuda and (not cached or (v.dtype is dtype and v.device == device and v.dim() == 3)))
    except (AttributeError, TypeError, ValueError):
        good = False
    if not good:
        _refuse_heads(q=q, k=k, **({"v": v} if cached else {}))
        raise ValueError("unsupported arguments")
    if nk != n:
        raise ValueError("q and k must have the same tokens: dimensions do not match")
    positions = _index("positions", positions, torch.int32, (n,), device)
    try:
        half, = inv_freq.shape
        good = (inv_freq.dtype is torch.float32 and 0 < 2 * half <= d and inv_freq.get_device() == device.index
                and inv_freq.is_contiguous())
    except (AttributeError, ValueError):
        good = False
    if not good:
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype is not torch.float32:
            raise TypeError("inv_freq must be a float32 tensor")
        if inv_freq.device != device:
            raise ValueError("inputs must be CUDA tensors on one device")
        raise ValueError(f"inv_freq must be a contiguous [rotary_dim / 2] with rotary_dim at most {d}, "
                         f"got {tuple(inv_freq.shape)}")
    q_token, q_head, unit = q.stride()
    if unit != 1:
        q = q.contiguous()
        q_token, q_head, unit = q.stride()
    k_token, k_head, unit = k.stride()
    if unit != 1:
        k = k.contiguous()
        k_token, k_head, unit = k.stride()
    v_ptr = slots_ptr = kc = vc = kb = vb = bs = nb = v_token = v_head = 0
    if cached:
        if v.shape != k.shape:
            raise ValueError("k and v must have matching shapes")
        slots = _index("slots", slots, torch.int64, (n,), device)
        nb, _, bs, kb, vb = _check_caches(k_cache, v_cache, q, hk)
        v_token, v_head, unit = v.stride()
        if unit != 1:
            v = v.contiguous()
            v_token, v_head, unit = v.stride()
        v_ptr, slots_ptr, kc, vc = v.data_ptr(), slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    q_out = torch.empty_like(q, memory_format=_PLAIN)
    k_out = torch.empty_like(k, memory_format=_PLAIN) if return_k else None
    if n == 0:
        return q_out, k_out
    args = _lib.ROPE_ARGS(code, n, h, hk, d, 2 * half, 1 if interleaved else 0, bs, nb, scale,
                          q.data_ptr(), k.data_ptr(), v_ptr, q_token, q_head, k_token, k_head, v_token, v_head,
                          positions.data_ptr(), slots_ptr, inv_freq.data_ptr(), q_out.data_ptr(),
                          k_out.data_ptr() if return_k else 0, kc, vc, kb, vb)
    _call((_lib._lib or _lib.load()).svdmlp_rope, args, device, "rope")
    return q_out, k_out


def rope_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
               inv_freq: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, interleaved: bool = False,
               scale: float = 1.0, return_k: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotates q [N, Hq, D] and k [N, Hk, D] to `positions` (int32 [N]) and
    writes the rotated k, and v, into the paged cache at `slots` (int64 [N];
    page_step gives both).  Returns (q, k), k only with `return_k`.

    The first 2 * len(inv_freq) elements of a head turn: pairs (i, i + half), or
    neighbours when `interleaved`; `scale` multiplies what turns.  A token whose
    slot is negative is written nowhere; two tokens of one call must not share a
    slot."""
    return _rope(q, k, v, positions, slots, inv_freq, k_cache, v_cache, interleaved, scale, return_k)


def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
         interleaved: bool = False, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """rope_cache without a cache: returns the rotated (q, k)."""
    return _rope(q, k, None, positions, None, inv_freq, None, None, interleaved, scale, True)


# -------------------------------------------------------------------- paging
class PageStep(NamedTuple):
    slots: torch.Tensor        # int64 [num_tokens]: where each new token goes, -1: nowhere
    positions: torch.Tensor    # int32 [num_tokens]: its position in its request
    cu_seqlens: torch.Tensor   # int32 [batch + 1]: offsets of the requests' new tokens
    seq_lens: torch.Tensor     # int32 [batch]: tokens held after this step
    free_count: torch.Tensor   # int32 [1]: blocks left on the free list
    missing: torch.Tensor      # int32 [1]: blocks the free list could not give


def kv_cache(num_blocks: int, kv_heads: int, block_size: int, head_dim: int, *, dtype=torch.bfloat16,
             device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """(k_cache, v_cache) of one layer, zeroed: [num_blocks, kv_heads, block_size, head_dim]."""
    for name, value in (("num_blocks", num_blocks), ("kv_heads", kv_heads), ("block_size", block_size),
                        ("head_dim", head_dim)):
        ops._positive(name, value)
    both = torch.zeros((2, num_blocks, kv_heads, block_size, head_dim), dtype=dtype, device=device)
    return both[0], both[1]


def _check_pages(block_table, seq_lens, new_lens, free_blocks, free_count, block_size, num_tokens):
    """Raises what is wrong with page_step's arguments; the index tensors, contiguous."""
    if not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    if block_table.dim() != 2 or min(block_table.shape) <= 0 or block_table.stride(1) != 1:
        raise ValueError(f"block_table must be a nonempty row-major [batch, width], got {tuple(block_table.shape)}")
    if not block_table.is_cuda:
        raise ValueError("block_table must be a CUDA tensor (the B200 path has no CPU fallback)")
    device = block_table.device
    b = block_table.shape[0]
    seq_lens = _index("seq_lens", seq_lens, torch.int32, (b,), device)
    new_lens = _index("new_lens", new_lens, torch.int32, (b,), device)
    free_count = _index("free_count", free_count, torch.int32, (1,), device)
    if not isinstance(free_blocks, torch.Tensor) or free_blocks.dtype != torch.int32:
        raise TypeError("free_blocks must be an int32 tensor")
    if free_blocks.dim() != 1 or not free_blocks.is_contiguous() or free_blocks.device != device:
        raise ValueError("free_blocks must be a contiguous 1D tensor on the table's device")
    ops._positive("block_size", block_size)
    if isinstance(num_tokens, bool) or not isinstance(num_tokens, int) or num_tokens < 0:
        raise ValueError(f"num_tokens must be a nonnegative integer, got {num_tokens}")
    return seq_lens, new_lens, free_count


def page_step(block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_blocks: torch.Tensor,
              free_count: torch.Tensor, block_size: int, num_tokens: int) -> PageStep:
    """Block tables, slots and positions of one forward pass from request lengths.

    Request b holds seq_lens[b] tokens and adds new_lens[b] (int32 [B]).  The
    blocks that it lacks come off the end of free_blocks[:free_count] (int32
    [F], int32 [1]), requests in order, and are entered into block_table [B, W]
    in place.  `num_tokens`, known to the caller, is at least the sum of
    new_lens; entries beyond it get slot -1.  The inputs other than
    block_table are left as they are: a caller keeps the returned seq_lens and
    free_count for the next step, and frees blocks by writing them behind
    free_count.  `missing` above zero means that the free list ran out: those
    blocks' entries and slots are -1.  A request's tokens beyond the table's
    W * block_size places get slot -1 too; they count in seq_lens, which tells
    them, and not in `missing`.  Negative lengths count as 0, and a request ends
    at 2^31 - 1 tokens."""
    try:
        b, width = block_table.shape
        index, one = block_table.get_device(), (1,)
        want = seq_lens.shape
        good = (index >= 0 and width > 0 and b > 0 and block_table.dtype is torch.int32 and block_table.stride(1) == 1
                and want == (b,) and seq_lens.dtype is torch.int32 and seq_lens.get_device() == index
                and new_lens.shape == want and new_lens.dtype is torch.int32 and new_lens.get_device() == index
                and free_count.shape == one and free_count.dtype is torch.int32 and free_count.get_device() == index
                and free_blocks.dtype is torch.int32 and free_blocks.get_device() == index and free_blocks.dim() == 1
                and seq_lens.is_contiguous() and new_lens.is_contiguous() and free_blocks.is_contiguous()
                and type(block_size) is int and block_size > 0 and type(num_tokens) is int and num_tokens >= 0)
    except (AttributeError, TypeError, ValueError):
        good = False
    if not good:
        seq_lens, new_lens, free_count = _check_pages(block_table, seq_lens, new_lens, free_blocks, free_count, block_size,
                                                      num_tokens)
        b, width = block_table.shape
    device = block_table.device
    slots = torch.empty(num_tokens, dtype=torch.int64, device=device)
    whole = torch.empty(num_tokens + 2 * b + 3, dtype=torch.int32, device=device)
    at = whole.data_ptr()
    positions, cu, lens, left, missing = whole.split_with_sizes((num_tokens, b + 1, b, 1, 1))
    cu_at = at + 4 * num_tokens
    lens_at = cu_at + 4 * (b + 1)
    left_at = lens_at + 4 * b
    args = _lib.PAGES_ARGS(b, num_tokens, block_size, width, free_blocks.shape[0], 0, block_table.data_ptr(),
                           block_table.stride(0), seq_lens.data_ptr(), new_lens.data_ptr(), free_blocks.data_ptr(),
                           free_count.data_ptr(), slots.data_ptr(), at, cu_at, lens_at, left_at, left_at + 4)
    _call((_lib._lib or _lib.load()).svdmlp_page_step, args, device, "page_step")
    return PageStep(slots, positions, cu, lens, left, missing)


def tree_positions(step: PageStep, tree_mask: torch.Tensor) -> torch.Tensor:
    """Positions (int32 [num_tokens]) of drafted trees, from a step's successive
    ones.

    A token of a tree follows its parent, not the token packed before it: its
    position is the context's length and its depth, the number of its ancestors,
    which are the bits of tree_mask (int64 [num_tokens], as tree_attention takes
    it) below its own.  Siblings share a position; the slots stay successive.
    Where the mask is a chain's the positions are the step's own."""
    cu, device = step.cu_seqlens, step.positions.device
    n = step.positions.shape[0]
    tree_mask = _index("tree_mask", tree_mask, torch.int64, (n,), device)
    token = torch.arange(n, dtype=torch.int32, device=device)
    request = torch.searchsorted(cu[1:], token, right=True).clamp_(max=cu.shape[0] - 2)
    node = token - cu[request]
    bit = torch.arange(_MASK_BITS, device=device)
    ancestors = ((tree_mask[:, None] >> bit) & 1) * (bit < node[:, None])
    depth = ancestors.sum(1, dtype=torch.int32)
    # tokens beyond the step's last are nobody's
    return torch.where(token < cu[-1], step.positions - node + depth, step.positions)


# ----------------------------------------------------------------- attention
def _group(q: torch.Tensor, kv_heads: int) -> None:
    if q.shape[1] % kv_heads:
        raise ValueError(f"{q.shape[1]} query heads are no multiple of {kv_heads} key/value heads")
    if q.shape[2] not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {q.shape[2]}")


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: Optional[torch.Tensor] = None, *, causal: bool = True, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v over packed sequences: q [Nq, Hq, D], k and v
    [Nk, Hk, D], sequence b the rows cu_q[b] .. cu_q[b + 1] and the keys cu_k[b]
    .. cu_k[b + 1] (int32 [B + 1] on the device; cu_k defaults to cu_q).  When
    causal, the queries are the last tokens of their sequence: query i of n
    sees the first m - n + i + 1 of m keys.  Rows that see no key, and rows of
    no sequence, give zeros.  `scale` defaults to 1 / sqrt(D).  bf16 or fp16,
    D 64 or 128; the probabilities are rounded to the inputs' type for the
    product with v, statistics and sums are fp32."""
    try:
        nq, h, d = q.shape
        nk, hk, dk = k.shape
        device, dtype = q.device, q.dtype
        code = _DTYPES.get(dtype)
        good = (code is not None and d == dk and (d == 128 or d == 64) and hk > 0 and h > 0 and h % hk == 0
                and v.shape == k.shape and k.dtype is dtype and v.dtype is dtype and q.is_cuda
                and k.device == device and v.device == device)
    except (AttributeError, TypeError, ValueError):
        good = False
    if not good:
        _refuse_heads(q=q, k=k, v=v)
        if k.shape != v.shape:
            raise ValueError("k and v must have matching shapes")
        _group(q, k.shape[1])
        raise ValueError("unsupported arguments")
    cu_q = _offsets("cu_q", cu_q, device)
    if cu_k is None:
        if nq != nk:
            raise ValueError("without cu_k, q and k must have the same tokens: dimensions do not match")
        cu_k = cu_q
    else:
        cu_k = _offsets("cu_k", cu_k, device)
        if cu_k.shape != cu_q.shape:
            raise ValueError("cu_q and cu_k must have matching shapes")
    scale = _scale(scale, d)
    given = out is not None
    out = _output(out, q) if given else torch.empty_like(q, memory_format=_PLAIN)
    if nq == 0:
        return out
    if nk == 0:
        return out.zero_()
    q, k, v = _rows(q), _rows(k), _rows(v)
    if given:
        _apart(out, q, k, v)
    ws = _workspace(device, d)
    q_token, q_head, _ = q.stride()
    k_token, k_head, _ = k.stride()
    v_token, v_head, _ = v.stride()
    o_token, o_head, _ = out.stride()
    args = _lib.PROMPT_ARGS(code, cu_q.shape[0] - 1, nq, nk, h, hk, d, 1 if causal else 0, scale, 0, q.data_ptr(),
                            k.data_ptr(), v.data_ptr(), q_token, q_head, k_token, k_head, v_token, v_head,
                            cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(), o_token, o_head, ws.ptr, ws.nbytes)
    _call((_lib._lib or _lib.load()).svdmlp_prompt_attention, args, device, "prompt_attention")
    return out


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, cu_q: torch.Tensor, *, max_tree: int,
                   tree_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of each request's newest tokens over the paged cache, which
    already holds their keys and values (rope_cache wrote them).

    q [N, Hq, D]; request b has the rows cu_q[b] .. cu_q[b + 1] (int32 [B + 1]),
    n of them, and seq_lens[b] tokens (int32 [B]) in the blocks block_table[b]
    names (int32 [B, W]); the newest n are its tree, in the rows' order.  Every
    row sees the seq_lens[b] - n tokens of the context.  In the tree, row i sees
    token j when bit j of tree_mask[row] (int64 [N]: a token's ancestors and
    itself) is set; without a mask, when j <= i, so n = 1 is ordinary decoding
    and a chain needs no mask.  `max_tree` is the largest n expected: it sizes
    the tiles, and larger trees are still computed, but a mask names the first
    64 tokens only, so with one max_tree is at most 64.  Rows that see
    nothing give zeros.  The block size is a power of two from 8 to 1024.  The
    keys of a tree that branches are turned to their depth (tree_positions)."""
    try:
        n, h, d = q.shape
        device, dtype = q.device, q.dtype
        code = _DTYPES.get(dtype)
        good = code is not None and h > 0 and d > 0 and q.is_cuda
    except (AttributeError, TypeError, ValueError):
        good = False
    if not good:
        _refuse_heads(q=q)
        raise ValueError("unsupported arguments")
    nb, hk, bs, kb, vb = _check_caches(k_cache, v_cache, q, None)
    if h % hk or (d != 128 and d != 64):
        _group(q, hk)
    if bs & (bs - 1) or not 8 <= bs <= 1024:
        raise ValueError(f"the cache's block size must be a power of two from 8 to 1024, got {bs}")
    cu_q = _offsets("cu_q", cu_q, device)
    b = cu_q.shape[0] - 1
    seq_lens = _index("seq_lens", seq_lens, torch.int32, (b,), device)
    if not isinstance(block_table, torch.Tensor) or block_table.dtype is not torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    if block_table.dim() != 2 or block_table.shape[0] != b or block_table.shape[1] <= 0 or block_table.stride(1) != 1:
        raise ValueError(f"block_table must be row-major [{b}, width], got {tuple(block_table.shape)}: "
                         "dimensions do not match")
    if block_table.device != device:
        raise ValueError("inputs must be CUDA tensors on one device")
    mask_ptr = 0
    if tree_mask is not None:
        tree_mask = _index("tree_mask", tree_mask, torch.int64, (n,), device)
        mask_ptr = tree_mask.data_ptr()
    ops._positive("max_tree", max_tree)
    if mask_ptr and max_tree > _MASK_BITS:
        raise ValueError(f"tree_mask names {_MASK_BITS} tokens of a request, max_tree is {max_tree}")
    scale = _scale(scale, d)
    given = out is not None
    out = _output(out, q) if given else torch.empty_like(q, memory_format=_PLAIN)
    if n == 0:
        return out
    q = _rows(q)
    if given:
        _apart(out, q, *(t.flatten(1).unsqueeze(1) for t in (k_cache, v_cache)))
    ws = _workspace(device, d)
    q_token, q_head, _ = q.stride()
    o_token, o_head, _ = out.stride()
    args = _lib.TREE_ARGS(code, b, n, h, hk, d, bs, nb, block_table.shape[1], max_tree, scale, 0, q.data_ptr(), q_token,
                          q_head, k_cache.data_ptr(), v_cache.data_ptr(), kb, vb, block_table.data_ptr(),
                          block_table.stride(0), seq_lens.data_ptr(), cu_q.data_ptr(), mask_ptr, out.data_ptr(), o_token,
                          o_head, ws.ptr, ws.nbytes)
    _call((_lib._lib or _lib.load()).svdmlp_tree_attention, args, device, "tree_attention")
    return out
