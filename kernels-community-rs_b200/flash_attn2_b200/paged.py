"""Operators around a paged K/V cache, on torch tensors: rotary positions with several axes, the append of new tokens,
attention of the newest tokens, and the eviction of tokens by the attention that they got.

The cache is a pool of pages, ``k_cache`` and ``v_cache`` [pages, page_size, Hk, D] (float16 or bfloat16, any page size, D a
multiple of 8 up to 256, any outer strides that are multiples of 8 elements), and an int32 ``block_table`` [B, pages of a
sequence]: token t of sequence b lies in row ``t % page_size`` of page ``block_table[b, t // page_size]``. ``seqlens_k`` (int32
[B], on the device) counts the tokens that the cache holds. Nothing is read back to the host, so that every call can be
captured in a CUDA graph, once a first call on the device has been made outside of one. Table entries and lengths are checked
on the device (and are not to be written while a call reads them): a page that is not in the pool is neither read nor written
and its keys are seen by nobody, a length that the table has no room for is cut, and ``cabi_ops.device_status()`` is 100 or 101
from then on until it is read.

A decoding step: ``q = paged_append(...)``, then ``paged_fwd`` with the lengths that count the new tokens, and now and then
``paged_evict``; all three with the same ``attn_mass`` where tokens are to be evicted. Prefill and training turn queries and
keys with ``rotary_axes_func`` and attend with ``flash_attn_func`` or ``flash_attn_varlen_func``.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
from pathlib import Path


def _load_native():
    path = Path(__file__).resolve().parent.parent / "lib" / "_fa2_paged.so"
    if not path.exists():
        raise ImportError(f"{path} is missing: build it with `python kernels-community-rs_b200/build.py`")
    import torch  # noqa: F401  (its libraries)

    loader = importlib.machinery.ExtensionFileLoader("_fa2_paged", str(path))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_fa2_paged", loader))
    loader.exec_module(module)
    return module


_native = _load_native()


def rotary_axes_func(q, k, positions, inv_freq, sections, interleaved_axes=False, interleaved_pairs=False):
    """Queries and keys turned by positions of several axes (time, height, width), with their gradients: (q_out, k_out).

    ``q`` [B, S, H, D] and ``k`` [B, S, Hk, D], or packed [T, H, D] and [T, Hk, D]; either may be None. ``positions`` [axes, B,
    S] (packed [axes, T]), int32 or int64; ``inv_freq`` float32, one frequency for each pair; ``sections`` says how many
    pairs each of the 1 to 4 axes has. A head's first ``2 * sum(sections)`` elements are turned, the others copied: pair i
    is the elements i and i + sum(sections), with ``interleaved_pairs`` 2 i and 2 i + 1. The first sections[0] pairs belong to
    axis 0, the next to axis 1 and so on; with ``interleaved_axes`` the axes take turns, pair i belonging to axis ``i % axes``
    while ``i < axes * sections[i % axes]`` and to axis 0 behind that. Angles are exact to a few 1e-7 rad
    at any position below 2^31 (frequencies up to 1)."""
    return _native.rotary(q, k, positions, inv_freq, sections, interleaved_axes, interleaved_pairs)


def paged_append(q, k, v, k_cache, v_cache, block_table, seqlens_k, positions, inv_freq, sections, interleaved_axes=False,
                 interleaved_pairs=False, cu_seqlens=None, seqlens_new=None, attn_mass=None):
    """New tokens: returns q turned, and puts k, turned, and v into the cache behind the ``seqlens_k`` tokens that each
    sequence has there (``seqlens_k`` is not changed). One launch.

    Dense: q [B, S, H, D], k and v [B, S, Hk, D]; with ``seqlens_new`` (int32 [B]) only the first rows of each sequence are
    tokens. Packed: [T, H, D] and [T, Hk, D] with ``cu_seqlens`` (int32 [B + 1]). Rows that are no tokens go nowhere. ``q``
    may be None. With ``attn_mass`` (see ``paged_fwd``) the new tokens' entries are set to 0: pages are used again, and a row
    keeps the weight of the token that lay there before. The other arguments are those of ``rotary_axes_func``. There is no
    gradient."""
    return _native.append(q, k, v, k_cache, v_cache, block_table, seqlens_k, positions, inv_freq, sections, interleaved_axes,
                          interleaved_pairs, cu_seqlens, seqlens_new, attn_mass)


def paged_fwd(q, k_cache, v_cache, block_table, seqlens_k, out=None, attn_mass=None, softmax_scale=None, window_size_left=-1,
              softcap=0.0, max_seqlen_k=None):
    """Attention of each sequence's last Sq tokens, which the cache holds already, over its pages: (out, LSE [B, H, Sq]).

    ``q`` [B, Sq, H, D] with at most 128 query rows per kv head (Sq * H / Hk). Token i of them sees the keys up to itself, and
    with ``window_size_left`` >= 0 no more than that many before it. A longer chunk of a prompt, once it is in the cache, goes in
    pieces: rows [i, j) of a chunk of S with ``seqlens_k - S + j``. A row without keys gives 0 and an LSE of +inf. The work
    is divided evenly over the SMs whatever the lengths are; a call repeats itself bit for bit, the ``attn_mass`` of pages
    that sequences share excepted (it is added in the order of arrival).

    ``attn_mass`` (float32 [pages, Hk, page_size], contiguous): each key's weights, summed over the query rows of its kv head,
    are added to its entry, which ``paged_append`` has started at 0 when it is given ``attn_mass`` too (a caller who does not
    give it sets the entries of new tokens to 0 before the first call that adds to them). This takes scratch memory of 4 bytes for
    each head, query and key, counted with ``max_seqlen_k`` where that is given (a bound on ``seqlens_k``; longer sequences are
    cut to it), else with all that the table has room for. There is no gradient."""
    return _native.fwd(q, k_cache, v_cache, block_table, seqlens_k, out, attn_mass, softmax_scale, window_size_left, softcap,
                       max_seqlen_k)


def paged_evict(k_cache, v_cache, attn_mass, block_table, seqlens_k, dst_block_table, budget, recent=0):
    """Eviction by accumulated weight: (new lengths int32 [B], kept int32 [B, Hk, budget]).

    Every kv head of a sequence with more than ``budget`` tokens keeps its newest ``recent`` tokens and, of the others, the
    ``budget - recent`` with the largest ``attn_mass`` (of equal ones the earlier; NaN counts as the largest); shorter
    sequences keep all. The rows that are kept, with their ``attn_mass``, go in their order to the pages of
    ``dst_block_table`` (int32 [B, pages]): pages of the same pool that ``block_table`` does not name, each named once. The old
    pages stay as they are. ``kept`` lists the old places of each head's rows, -1 behind the last. Keys carry their rotary
    positions with them; places in the cache are no longer positions."""
    return _native.evict(k_cache, v_cache, attn_mass, block_table, seqlens_k, dst_block_table, budget, recent)
