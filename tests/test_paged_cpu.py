"""CPU: the index arithmetic of the operators on a paged cache (csrc/paged_index.h) through a small library around that header, and
what their C entry points refuse before anything runs."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent

SHIM = r'''
#include <cuda_runtime.h>
#include "paged_index.h"
using namespace fa2;
extern "C" {
int fast_div(int n, int d) { return make_div(d).div(n); }
int fast_mod(int n, int d) { return make_div(d).mod(n); }
int page_of(const int32_t* pages, int64_t stride, int max_pages, int num_pages, int page_size, int b, int slot) {
  PageTable t;
  t.pages = pages; t.stride = stride; t.max_pages = max_pages; t.num_pages = num_pages; t.page_size = make_div(page_size);
  return t.page_of(b, slot);
}
int cut(int n, int64_t most) { return cut_length(n, most); }
int first_tile(int n, int sq, int window, int tile) { return first_seen_tile(n, sq, window, tile); }
int tiles(int n, int sq, int window, int tile) { return tiles_of(n, sq, window, tile); }
int64_t begin(int64_t c, int64_t tiles, int64_t grid) { return share_begin(c, tiles, grid); }
int owner(int64_t tile, int64_t tiles, int64_t grid) { return share_owner(tile, tiles, grid); }
int axis(int i, int axes, const int32_t* sections, int turns) { return axis_of_pair(i, axes, sections, turns); }
}
'''


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "shim.cc").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{ROOT / 'kernels-community-rs_b200' / 'csrc'}",
                    "-I/usr/local/cuda/include", str(d / "shim.cc"), "-o", str(d / "shim.so")], check=True)
    lib = C.CDLL(str(d / "shim.so"))
    lib.begin.restype = C.c_int64
    lib.begin.argtypes = [C.c_int64] * 3
    lib.owner.argtypes = [C.c_int64] * 3
    lib.cut.argtypes = [C.c_int, C.c_int64]
    return lib


def test_division_by_multiplication(index):
    rng = random.Random(1)
    divisors = [1, 2, 3, 5, 7, 16, 17, 48, 100, 255, 256, 641, 65535, 65536, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1]
    for d in divisors + [rng.randrange(1, 2 ** 31) for _ in range(200)]:
        around = [k * d + e for k in (0, 1, 2, (2 ** 31 - 1) // d) for e in (-1, 0, 1)]
        for n in around + [2 ** 31 - 1, 2 ** 31 - 2] + [rng.randrange(2 ** 31) for _ in range(50)]:
            if 0 <= n < 2 ** 31:
                assert index.fast_div(n, d) == n // d and index.fast_mod(n, d) == n % d, (n, d)


def test_pages_that_cannot_be_are_none(index):
    """Entries outside the pool, and tokens outside the table's row, give no page; nothing behind the row is read."""
    table = (C.c_int32 * 8)(3, -1, 7, 2 ** 31 - 1, 0, 8, -2 ** 31, 5)

    def page(b, slot):
        return index.page_of(table, C.c_int64(4), 4, 8, 10, b, slot)

    assert [page(0, s) for s in (0, 9, 10, 20, 39)] == [3, 3, -1, 7, -1]
    assert [page(1, s) for s in (0, 10, 29, 30)] == [0, -1, -1, 5]
    assert [page(0, s) for s in (-1, -2 ** 31, 40, 2 ** 31 - 1)] == [-1] * 4
    # a row of a table with room for more than 2^31 tokens
    assert index.page_of(table, C.c_int64(4), 4, 8, 2 ** 30, 0, 2 ** 31 - 1) == -1
    assert index.page_of(table, C.c_int64(4), 4, 8, 2 ** 30, 0, 2 ** 30 - 1) == 3


def test_lengths_are_cut(index):
    assert [index.cut(n, 100) for n in (-2 ** 31, -1, 0, 100, 101, 2 ** 31 - 1)] == [0, 0, 0, 100, 100, 100]
    assert index.cut(2 ** 31 - 1, 2 ** 40) == 2 ** 31 - 1


@pytest.mark.parametrize("tile", [64, 128])
def test_tiles_hold_every_key_that_a_row_sees(index, tile):
    for n in (0, 1, 63, 64, 65, 127, 128, 129, 1000, 4096, 2 ** 31 - 70000):
        for sq in (1, 2, 5, 128):
            for window in (-1, 0, 1, 63, 64, 500, 2 ** 31 - 70001):
                first, count = index.first_tile(n, sq, window, tile), index.tiles(n, sq, window, tile)
                lo = max(0, n - sq - window) if window >= 0 else 0
                assert count >= 1 and first * tile <= lo and (lo - first * tile < tile)
                assert (first + count) * tile >= n
                if n > first * tile:
                    assert (first + count - 1) * tile < n


def test_shares_cover_the_tiles_once(index):
    rng = random.Random(2)
    for tiles, grid in [(1, 1), (1, 148), (147, 148), (148, 148), (149, 148), (5000, 148), (7, 3)] + \
            [(rng.randrange(1, 3000), rng.randrange(1, 149)) for _ in range(50)]:
        bounds = [index.begin(c, tiles, grid) for c in range(grid + 1)]
        assert bounds[0] == 0 and bounds[-1] == tiles and sorted(bounds) == bounds
        if tiles >= grid:  # the kernel takes no more CTAs than tiles: then each has some, and a unit's parts are neighbours'
            assert all(a < b for a, b in zip(bounds, bounds[1:]))
        for x in range(tiles):
            c = index.owner(x, tiles, grid)
            assert bounds[c] <= x < bounds[c + 1], (x, tiles, grid)
    # long lists: products past 32 bits
    tiles, grid = 2 ** 40 + 12345, 148
    for c in (0, 1, 77, 147):
        assert index.owner(index.begin(c, tiles, grid), tiles, grid) == c
        assert index.owner(index.begin(c + 1, tiles, grid) - 1, tiles, grid) == c


@pytest.mark.parametrize("sections", [(64,), (16, 24, 24), (24, 20, 20), (1, 0, 2, 1), (0, 5), (43, 21, 0)])
def test_axes_of_the_pairs(index, sections):
    n, axes = sum(sections), len(sections)
    s = (C.c_int32 * 4)(*sections)
    assert [index.axis(i, axes, s, 0) for i in range(n)] == [a for a, c in enumerate(sections) for _ in range(c)]
    want = [0] * n
    for a in range(1, axes):
        want[a:axes * sections[a]:axes] = [a] * len(range(a, min(n, axes * sections[a]), axes))
    assert [index.axis(i, axes, s, 1) for i in range(n)] == want


# ---------------------------------------------------------------- the C entry points
def _cache(**kw):
    from flash_attn2_b200 import _cabi

    c = _cabi.PagedCache(size=C.sizeof(_cabi.PagedCache), k=1 << 20, v=1 << 21, k_stride=(16 * 2 * 64, 2 * 64, 64),
                         v_stride=(16 * 2 * 64, 2 * 64, 64), attn_mass=1 << 22, block_table=1 << 23, block_table_stride=4,
                         seqlens_k=1 << 24, num_pages=8, page_size=16, max_pages=4, batch=2, heads_k=2, head_dim=64, dtype=_cabi.FA2_BF16)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def _turn(**kw):
    from flash_attn2_b200 import _cabi

    a = _cabi.RotaryArgs(size=C.sizeof(_cabi.RotaryArgs), q=1 << 20, q_out=1 << 21, k=1 << 22, k_out=1 << 23, positions=1 << 24,
                         inv_freq=1 << 25, position_bits=64, dtype=_cabi.FA2_BF16, batch=2, seqlen=3, heads=4, heads_k=2, head_dim=64,
                         axes=3, sections=(12, 10, 10))
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def _fwd(cache=None, **kw):
    from flash_attn2_b200 import _cabi

    a = _cabi.PagedFwdArgs(size=C.sizeof(_cabi.PagedFwdArgs), cache=C.pointer(_cache() if cache is None else cache), q=1 << 20, out=1 << 21,
                           lse=1 << 22, q_stride=(256, 256, 64), o_stride=(256, 256, 64), seqlen_q=1, heads=4, softmax_scale=0.1,
                           window_left=-1)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def _refused(function, args, code, word, *more):
    from flash_attn2_b200 import _cabi

    lib = _cabi.load()
    assert getattr(lib, function)(C.byref(args), *more) == code, lib.fa2_last_error()
    assert word in lib.fa2_last_error().decode()


BAD_CACHES = [(dict(size=8), -1, "size"), (dict(dtype=7), -2, "float16"), (dict(head_dim=60), -1, "head dim"), (dict(head_dim=264), -1, "head dim"),
              (dict(num_pages=0), -1, "positive"), (dict(page_size=-1), -1, "positive"), (dict(max_pages=0), -1, "positive"),
              (dict(batch=70000), -1, "65535"), (dict(heads_k=0), -1, "65535"), (dict(k=0), -1, "non-null"), (dict(block_table=0), -1, "non-null"),
              (dict(k=(1 << 20) + 8), -1, "aligned"), (dict(v_stride=(2048, 100, 64)), -1, "multiples of 8"),
              (dict(block_table=(1 << 20) + 2), -1, "4-byte"), (dict(seqlens_k=(1 << 20) + 1), -1, "4-byte"), (dict(attn_mass=(1 << 20) + 3), -1, "4-byte"),
              (dict(k_stride=(2048, -128, 64)), -1, "negative"), (dict(reserved=1), -1, "reserved")]


@pytest.mark.parametrize("change,code,word", BAD_CACHES, ids=[str(c[0]) for c in BAD_CACHES])
def test_bad_caches_are_refused(built_libs, change, code, word):
    from flash_attn2_b200 import _cabi

    cache = _cache(**change)
    _refused("fa2_paged_fwd", _fwd(cache), code, word, None, 0, None)
    evict = _cabi.PagedEvictArgs(size=C.sizeof(_cabi.PagedEvictArgs), cache=C.pointer(cache), dst_block_table=1 << 20, dst_max_pages=1,
                                 budget=4, seqlens_out=1 << 20, kept=1 << 20)
    _refused("fa2_paged_evict", evict, code, word, None)
    append = _cabi.PagedAppendArgs(size=C.sizeof(_cabi.PagedAppendArgs), turn=C.pointer(_turn()), cache=C.pointer(cache), v=1 << 20)
    _refused("fa2_paged_append", append, code, word, None)


BAD_TURNS = [(dict(size=8), -1, "size"), (dict(dtype=9), -2, "float16"), (dict(head_dim=12), -1, "head dim"), (dict(axes=0), -1, "axes"),
             (dict(axes=5), -1, "axes"), (dict(sections=(40, 1, 1)), -1, "sections"), (dict(sections=(0, 0, 0)), -1, "sections"),
             (dict(sections=(-1, 9, 9)), -1, "sections"), (dict(sections=(2, 10, 10), interleaved_axes=1), -1, "turns"),
             (dict(position_bits=16), -1, "position_bits"), (dict(positions=0), -1, "positions"), (dict(positions=(1 << 20) + 4), -1, "aligned"),
             (dict(inv_freq=0), -1, "inv_freq"), (dict(q_out=0), -1, "q_out"), (dict(q=(1 << 20) + 1), -1, "aligned"),
             (dict(batch=2 ** 20, seqlen=2 ** 12), -1, "batch"), (dict(heads=0), -1, "heads"), (dict(k_out=0), -1, "k_out"),
             (dict(seqlen=-1), -1, "batch")]


@pytest.mark.parametrize("change,code,word", BAD_TURNS, ids=[str(c[0]) for c in BAD_TURNS])
def test_bad_turns_are_refused(built_libs, change, code, word):
    _refused("fa2_rotary", _turn(**change), code, word, None)


@pytest.mark.parametrize("change,code,word", [
    (dict(turn=dict(heads_k=4)), -1, "cache's heads"), (dict(turn=dict(head_dim=72)), -1, "cache's heads"), (dict(turn=dict(dtype=0)), -2, "dtype"),
    (dict(turn=dict(k=0)), -1, "k is null"), (dict(turn=dict(batch=3)), -1, "batch"), (dict(cu_seqlens=1 << 20), -1, "cu_seqlens"), (dict(seqlens_new=(1 << 20) + 2), -1, "4-byte"),
    (dict(v=0), -1, "v must"), (dict(v=(1 << 20) + 1), -1, "v must"), (dict(size=8), -1, "size")], ids=str)
def test_bad_appends_are_refused(built_libs, change, code, word):
    from flash_attn2_b200 import _cabi

    change = dict(change)
    turn, cache = _turn(**change.pop("turn", {})), _cache()
    a = _cabi.PagedAppendArgs(size=C.sizeof(_cabi.PagedAppendArgs), turn=C.pointer(turn), cache=C.pointer(cache), v=1 << 20)
    for name, value in change.items():
        setattr(a, name, value)
    _refused("fa2_paged_append", a, code, word, None)


@pytest.mark.parametrize("change,word", [
    (dict(size=8), "size"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"), (dict(seqlen_q=-1), "seqlen_q"), (dict(seqlen_q=65), "128 query rows"),
    (dict(softmax_scale=float("nan")), "softmax_scale"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap"),
    (dict(max_seqlen_k=-1), "max_seqlen_k"), (dict(q=0), "non-null"), (dict(out=0), "non-null"), (dict(lse=0), "non-null"), (dict(lse=(1 << 20) + 2), "4-byte"),
    (dict(q=(1 << 20) + 2), "aligned"), (dict(o_stride=(256, 256, 60)), "multiples of 8")], ids=str)
def test_bad_forwards_are_refused(built_libs, change, word):
    _refused("fa2_paged_fwd", _fwd(**change), -1, word, None, 0, None)


@pytest.mark.parametrize("change,word", [
    (dict(size=8), "size"), (dict(budget=0), "budget"), (dict(budget=2 ** 31 - 1), "budget"), (dict(kept=(1 << 20) + 1), "4-byte"), (dict(recent=-1), "recent"), (dict(recent=5), "recent"), (dict(dst_block_table=0), "dst_block_table"),
    (dict(dst_max_pages=0), "dst_block_table"), (dict(kept=0), "kept"), (dict(seqlens_out=0), "seqlens_out"), (dict(reserved=1), "reserved")], ids=str)
def test_bad_evictions_are_refused(built_libs, change, word):
    from flash_attn2_b200 import _cabi

    cache = _cache()
    a = _cabi.PagedEvictArgs(size=C.sizeof(_cabi.PagedEvictArgs), cache=C.pointer(cache), dst_block_table=1 << 20, dst_max_pages=1, budget=4,
                             recent=1, seqlens_out=1 << 20, kept=1 << 20)
    for name, value in change.items():
        setattr(a, name, value)
    _refused("fa2_paged_evict", a, -1, word, None)
    without = _cache(attn_mass=None)
    b = _cabi.PagedEvictArgs(size=C.sizeof(_cabi.PagedEvictArgs), cache=C.pointer(without), dst_block_table=1 << 20, dst_max_pages=1, budget=4,
                             seqlens_out=1 << 20, kept=1 << 20)
    _refused("fa2_paged_evict", b, -1, "attn_mass", None)


def test_null_arguments_are_refused(built_libs):
    from flash_attn2_b200 import _cabi

    lib = _cabi.load()
    assert lib.fa2_rotary(None, None) == lib.fa2_paged_append(None, None) == lib.fa2_paged_evict(None, None) == -1
    assert lib.fa2_paged_fwd(None, None, 0, None) == -1 and lib.fa2_paged_fwd_workspace_bytes(None) == 0


@pytest.mark.parametrize("struct,mirror", [("fa2_paged_cache", "PagedCache"), ("fa2_rotary_args", "RotaryArgs"),
                                           ("fa2_paged_append_args", "PagedAppendArgs"), ("fa2_paged_fwd_args", "PagedFwdArgs"),
                                           ("fa2_paged_evict_args", "PagedEvictArgs")])
def test_ctypes_mirrors_follow_the_header(struct, mirror, tmp_path):
    from flash_attn2_b200 import _cabi
    from tests.test_boundary_cpu import _header_fields

    cls = getattr(_cabi, mirror)
    assert [(n, [str(t._length_)] if hasattr(t, "_length_") else []) for n, t in cls._fields_] == _header_fields(struct)
    names = [n for n, _ in cls._fields_]
    (tmp_path / "p.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fa2_b200.h"\nint main(){printf("%zu", sizeof(' + struct + "));" +
                                  "".join(f'printf(" %zu", offsetof({struct}, {n}));' for n in names) + "return 0;}")
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(cls)] + [getattr(cls, n).offset for n in names]


def test_cpu_tensors_and_wrong_types_are_refused(built_libs):
    import flash_attn2_b200 as fa

    z = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    pos, freq, table, n = torch.zeros(1, 1, 3, dtype=torch.int32), torch.zeros(32), torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    cache, mass = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 16)
    calls = [lambda: fa.rotary_axes_func(z, z, pos, freq, (32,)),
             lambda: fa.paged_append(z, z, z, cache, cache.clone(), table, n, pos, freq, (32,)),
             lambda: fa.paged_fwd(z, cache, cache, table, n), lambda: fa.paged_evict(cache, cache, mass, table, n, table, 4)]
    for call in calls:
        with pytest.raises(NotImplementedError):
            call()
    with pytest.raises(TypeError):
        fa.rotary_axes_func(z, z, pos, freq, 32)
    with pytest.raises(TypeError):
        fa.rotary_axes_func(z, z, pos, freq, (32.0,))
    with pytest.raises(TypeError):
        fa.paged_fwd("q", cache, cache, table, n)
    with pytest.raises(ValueError):
        fa.rotary_axes_func(z, z, pos, freq, (1, 2, 3, 4, 5))
    with pytest.raises(ValueError):
        fa.rotary_axes_func(None, None, pos, freq, (32,))
    with pytest.raises(TypeError):
        fa.paged_evict(cache, cache, mass, table, n, table, 4.0)


# ---------------------------------------------------------------- what the kernels' source has to say
def _kernels_with_barriers():
    """(file, name, body from the barriers' set-up on) of each kernel that sets up mbarriers."""
    import re

    for path in sorted((ROOT / "kernels-community-rs_b200" / "csrc").glob("*.cu")):
        for kernel in re.split(r"^(?=__global__ )", path.read_text(), flags=re.M)[1:]:
            kernel = kernel[:kernel.index("\n}\n")]
            if "mbar_init(" in kernel:
                yield path.name, re.search(r"\b(\w+_kernel)\(", kernel)[1], kernel[kernel.rindex("mbar_fence_init()"):]


def test_barriers_and_abort_words_are_seen_by_all_warps_before_their_first_wait():
    """A block barrier that no condition guards (two spaces deep) stands between the set-up of a kernel's mbarriers and abort word and
    the first wait. What a missing one does depends on the warps' timing, so that no run would show it."""
    import re

    found = list(_kernels_with_barriers())
    assert {"fwd_paged_kernel", "fwd_kernel", "fwd_decode_kernel", "bwd_kernel"} <= {name for _, name, _ in found}
    for path, name, body in found:
        barrier = re.search(r"^  __syncthreads\(\);", body, flags=re.M)
        assert barrier is not None, (path, name)
        assert not re.search(r"(warp|mbar)_wait", body[:barrier.start()]), (path, name)


LIST_SHIM = r'''
#include <cuda_runtime.h>
#include "paged_index.h"
extern "C" int there(int first, int n, int grid) { return fa2::parts_there(first, n, grid); }
extern "C" int place(int larger, int ties, int most_ties, int wanted) { return fa2::list_place(larger, ties, most_ties, wanted); }
'''


def _library(tmp_path, source):
    (tmp_path / "shim.cc").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=signed-integer-overflow", "-fsanitize-undefined-trap-on-error", "-shared", "-fPIC",
                    f"-I{ROOT / 'kernels-community-rs_b200' / 'csrc'}", "-I/usr/local/cuda/include", str(tmp_path / "shim.cc"), "-o",
                    str(tmp_path / "shim.so")], check=True)
    return C.CDLL(str(tmp_path / "shim.so"))


def test_parts_outside_the_workspace_are_none(tmp_path):
    """The join reads the slots of CTAs [first, first + n): whatever the workspace says, those that there are."""
    lib = _library(tmp_path, LIST_SHIM)
    words = (-2 ** 31, -2 ** 31 + 1, -1, 0, 1, 2, 146, 147, 148, 149, 2 ** 30, 2 ** 31 - 148, 2 ** 31 - 1)
    for grid in (1, 2, 148):
        for first in words:
            for n in words:
                assert bool(lib.there(first, n, grid)) == (0 <= first and n > 0 and first + n <= grid), (first, n, grid)


def test_the_join_and_the_weights_ask_for_the_parts_they_read():
    source = (ROOT / "kernels-community-rs_b200" / "csrc" / "fwd_paged_sm100.cu").read_text()
    for function in ("join_parts", "add_weights"):
        body = source[source.index(f" void {function}("):]
        body = body[:body.index("\n}\n")]
        assert -1 < body.find("parts_there(") < body.index("part_of("), function


def test_lists_of_kept_tokens_end_where_they_should(tmp_path):
    """The places of an eviction's list are those below `wanted`, each once, also where the weights that are counted last are not those
    that the border was found with (more keys above it than there were)."""
    place = _library(tmp_path, LIST_SHIM).place
    rng = random.Random(3)
    for _ in range(200):
        keys = [rng.randrange(6) for _ in range(rng.randrange(2, 60))]
        wanted = rng.randrange(1, len(keys))
        border = sorted(keys, reverse=True)[wanted - 1]
        ties = wanted - sum(k > border for k in keys)
        for seen in (keys, [k + rng.randrange(3) for k in keys], [9] * len(keys)):  # as they were, and grown meanwhile
            at_above = at_ties = 0
            places = []
            for k in seen:
                at = place(at_above, at_ties, ties, wanted)
                assert -1 <= at < wanted
                if at >= 0 and (k > border or (k == border and at_ties < ties)):
                    places.append(at)
                at_above += k > border
                at_ties += k == border
            assert len(set(places)) == len(places)
            if seen is keys:
                assert places == list(range(wanted))


def test_the_list_is_written_at_such_places():
    source = (ROOT / "kernels-community-rs_b200" / "csrc" / "paged_evict_sm100.cu").read_text()
    choice = source[source.index("done_above = 0"):source.index("kMoveThreads")]
    assert "kept[place] = " in choice and choice.count("kept[") == 1 and "place = list_place(" in choice


@pytest.mark.parametrize("name,dim", [("q", 0), ("q", 1), ("q", 2), ("k", 0), ("k", 1), ("k", 2)])
def test_turns_in_place_with_other_strides_are_refused(built_libs, name, dim):
    """In place is allowed where each element stays where it is: a stride of the output that differs would make it a race."""
    strides = [3 * 256, 256, 64]
    other = list(strides)
    other[dim] += 64
    args = dict(q_stride=strides, q_out_stride=strides, k_stride=strides, k_out_stride=strides)
    args[name + "_out_stride"] = other
    a = _turn(**{k: tuple(v) for k, v in args.items()})
    setattr(a, name + "_out", getattr(a, name))
    _refused("fa2_rotary", a, -1, f"{name}_out is {name}", None)


def test_tiles_of_the_kernels_size_hold_every_key_that_a_row_sees(index):
    """The kernel's tiles have 16 keys."""
    for n in list(range(0, 50)) + [127, 128, 129, 1000, 4093, 4096, 131071, 2 ** 31 - 70000]:
        for sq in (1, 2, 5, 17, 128):
            for window in (-1, 0, 1, 15, 16, 17, 63, 500, 2 ** 31 - 70001):
                first, count = index.first_tile(n, sq, window, 16), index.tiles(n, sq, window, 16)
                lo = max(0, n - sq - window) if window >= 0 else 0
                assert count >= 1 and first * 16 <= lo < first * 16 + 16
                assert (first + count) * 16 >= n
                assert n <= first * 16 or (first + count - 1) * 16 < n


@pytest.mark.parametrize("grid", [1, 2, 147, 148, 253, 254, 255, 256])
@pytest.mark.parametrize("tiles", [2 ** 24 - 2, 2 ** 24 - 1, 2 ** 24, 2 ** 24 + 1])
def test_shares_where_the_divisions_change_their_width(index, tiles, grid):
    """Up to 2^24 - 1 tiles and 254 CTAs the products stay below 2^32 (254 * (2^24 - 1) and what share_owner adds); beyond they have 64 bits."""
    index.begin.restype = C.c_int64
    bounds = [index.begin(c, tiles, grid) for c in range(grid + 1)]
    assert bounds == [c * tiles // grid for c in range(grid + 1)]
    for c in range(grid):
        for x in (bounds[c], bounds[c] + 1, (bounds[c] + bounds[c + 1]) // 2, bounds[c + 1] - 1):
            assert index.owner(x, tiles, grid) == c, (x, c)
