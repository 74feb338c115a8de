"""GPU: attention over a paged cache, the append of new tokens and the eviction against 64-bit arithmetic: lengths of 0 and 1, pages that
end inside tiles, every head-dim bucket, rows without keys, what lies in masked places, accumulated weights, graphs, streams, far offsets."""
import ctypes as C
import math
import subprocess
import sys

import pytest
import torch

from tests._paged import attend, choose, make_cache, rows_of, turn, turn_tolerance

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _table(t):
    return torch.tensor(t, dtype=torch.int32, device="cuda")


def _close(out, lse, want, dtype, v_cache, keys):
    """The output's own rounding; errors of the scores move the weights, and with them the values; P is the sum of two 16-bit numbers
    (2^-16 of it, in fp16 2^-25 of the largest of a row for each key)."""
    o_ref, lse_ref, _, delta = want
    v = v_cache.float().abs().nan_to_num(0, 0, 0).max().item()
    spread = 2 * delta + (2.0 ** -15 if dtype == torch.bfloat16 else 2.0 ** -21 + keys * 2.0 ** -25)
    torch.testing.assert_close(out.cpu().double(), o_ref, rtol=HALF[dtype] * 1.001, atol=spread * v + torch.finfo(dtype).tiny, equal_nan=True)
    torch.testing.assert_close(lse.cpu().double(), lse_ref, rtol=2 ** -22, atol=delta)


# lengths, h, hk, sq, d, page, options
CASES = [
    ([1], 1, 1, 1, 8, 1, {}),
    ([0, 1, 2], 4, 2, 1, 64, 16, {}),
    ([15, 16, 17, 31, 33], 8, 8, 1, 128, 16, {}),
    ([127, 128, 129, 1, 0, 255, 257], 32, 8, 1, 128, 64, {}),
    ([5000], 32, 8, 1, 128, 16, {}),
    ([1000, 77, 640], 16, 2, 1, 128, 48, {}),
    ([300, 4097, 12], 16, 1, 1, 96, 7, {}),                            # odd pages that end anywhere in a tile
    ([700, 3], 34, 2, 1, 72, 100, {}),                                 # 17 rows: two row tiles
    ([513, 64], 128, 1, 1, 64, 256, {}),                               # 128 rows
    ([900, 20, 1500], 12, 4, 1, 192, 32, {}),
    ([2049, 63, 65, 64], 8, 4, 1, 256, 128, {}),
    ([400], 4, 4, 1, 136, 16, {}),
    ([300, 2, 5, 0, 1], 16, 4, 4, 128, 16, {}),                        # rows without keys
    ([2000, 130], 8, 2, 17, 64, 16, {}),
    ([1300, 40], 8, 4, 5, 128, 64, dict(window=100)),
    ([1300, 40, 7], 8, 8, 1, 128, 64, dict(window=16)),
    ([500, 17], 6, 2, 3, 128, 48, dict(window=0)),
    ([3000], 8, 1, 2, 256, 16, dict(window=1500, softcap=20.0)),
    ([1000, 50], 8, 2, 1, 128, 16, dict(softcap=5.0)),
    ([200, 31], 4, 2, 2, 64, 16, dict(scale=-0.3)),
    ([64] * 300, 4, 2, 1, 64, 32, {}),                                 # more sequences than a CTA has threads
    ([(i * 37) % 400 for i in range(521)], 2, 1, 1, 64, 16, {}),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[1:]}")
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_attention(case, dtype):
    import flash_attn2_b200 as fa2

    lengths, h, hk, sq, d, page, opt = case
    layout = ("nhd", "hnd", "fused")[len(lengths) % 3]
    k, v, table = make_cache(1, lengths, hk, d, page, dtype, layout=layout)
    q = torch.randn(len(lengths), sq, h, d, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    want = attend(q, k, v, table, lengths, **opt)
    kw = dict(softmax_scale=opt.get("scale"), window_size_left=opt.get("window", -1), softcap=opt.get("softcap", 0.0))
    out, lse = fa2.paged_fwd(q, k, v, table, _table(lengths), **kw)
    assert fa2.cabi_ops.device_status() == 0
    _close(out, lse, want, dtype, v, max(lengths))
    again = fa2.paged_fwd(q, k, v, table, _table(lengths), **kw, max_seqlen_k=max(1, max(lengths)))
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    # accumulated weights
    mass = torch.rand(k.shape[0], hk, page, generator=torch.Generator().manual_seed(3)).cuda()
    before = mass.clone()
    with_mass = fa2.paged_fwd(q, k, v, table, _table(lengths), attn_mass=mass, **kw)
    assert torch.equal(with_mass[0], out) and torch.equal(with_mass[1], lse)
    expected = before.cpu().double()
    for b, (n, w) in enumerate(zip(lengths, want[2])):
        t = torch.arange(n)
        pages = table.cpu()[b].long()[t // page]
        expected[pages, :, t % page] += w.T
    # a weight is off by its score's error and its own roundings, the sum by its rounding
    torch.testing.assert_close(mass.cpu().double(), expected, rtol=2 ** -23, atol=2 * want[3] * sq * (h // hk))
    assert fa2.cabi_ops.device_status() == 0


@pytest.mark.parametrize("page", [16, 24, 9])
@pytest.mark.parametrize("d", [64, 104, 128, 192, 256])
@pytest.mark.parametrize("h,hk,sq", [(5, 1, 1), (12, 1, 1), (16, 2, 3), (18, 2, 5)])
def test_rows_dims_and_pages(page, d, h, hk, sq):
    """Units of 8, 16 and 32 rows and of more (5, 12, 24, 45 rows), every head-dim bucket, whole and broken tiles."""
    import flash_attn2_b200 as fa2

    lengths = [700, 65, 2, 0, 1300]
    k, v, table = make_cache(14, lengths, hk, d, page, torch.bfloat16)
    q = torch.randn(5, sq, h, d, generator=torch.Generator().manual_seed(15)).bfloat16().cuda()
    want = attend(q, k, v, table, lengths, window=600)
    mass = torch.zeros(k.shape[0], hk, page, device="cuda")
    out, lse = fa2.paged_fwd(q, k, v, table, _table(lengths), attn_mass=mass, window_size_left=600)
    assert fa2.cabi_ops.device_status() == 0
    _close(out, lse, want, torch.bfloat16, v, 700)
    for b, n in enumerate(lengths):
        got = mass[table[b].long().clamp(min=0)].transpose(1, 2).flatten(0, 1)[:n].T.cpu().double()
        torch.testing.assert_close(got, want[2][b], rtol=2 ** -23, atol=2 * want[3] * sq * (h // hk))


def test_scores_that_keep_growing():
    """Keys in the order of their scores, over a range of 2^150: the running maximum moves many times, and early weights vanish."""
    import flash_attn2_b200 as fa2

    n, d = 2000, 64
    k, v, table = make_cache(16, [n], 1, d, 16, torch.float16)
    q = torch.zeros(1, 2, 4, d, dtype=torch.float16, device="cuda")
    q[..., 0] = 8.0
    ramp = torch.linspace(-52, 52, n).half()
    for order in (ramp, ramp.flip(0)):
        t = torch.arange(n)
        k[table[0].long().cpu()[t // 16], t % 16, 0, 0] = order.cuda()
        want = attend(q, k, v, table, [n])
        out, lse = fa2.paged_fwd(q, k, v, table, _table([n]))
        _close(out, lse, want, torch.float16, v, n)


def test_heads_that_share_their_memory():
    """A cache whose heads are one, expanded."""
    import flash_attn2_b200 as fa2

    k, v, table = make_cache(17, [300, 40], 1, 128, 16, torch.bfloat16)
    q = torch.randn(2, 1, 8, 128, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    want = fa2.paged_fwd(q, k, v, table, _table([300, 40]))
    got = fa2.paged_fwd(q, k.expand(-1, -1, 4, -1), v.expand(-1, -1, 4, -1), table.expand(2, -1), _table([300, 40]))
    # the same products in units of other rows: the parts are cut elsewhere
    torch.testing.assert_close(got[0], want[0], rtol=2 ** -7, atol=1e-4)
    torch.testing.assert_close(got[1], want[1], rtol=0, atol=1e-5)


def test_inference_mode_and_parameters():
    import flash_attn2_b200 as fa2

    k, v, table = make_cache(18, [30], 2, 64, 16, torch.bfloat16)
    pos, freq = torch.full((1, 1, 1), 30, device="cuda"), torch.nn.Parameter(torch.rand(32, device="cuda"), requires_grad=False)
    with torch.inference_mode():
        x = torch.randn(1, 1, 2, 64, device="cuda").bfloat16()
        own = k.clone()
        q = fa2.paged_append(x, x, x, own, v.clone(), table, _table([30]), pos, freq, (32,))
        assert torch.equal(q, fa2.rotary_axes_func(x, None, pos, freq, (32,))[0])
        assert torch.equal(own[table[0, 1].long(), 14], q[0, 0])
        fa2.paged_fwd(q, own, v, table, _table([30]))


CAPTURE = r"""
import sys
sys.path[:0] = ["kernels-community-rs_b200"]
import torch
import flash_attn2_b200 as fa2
k = torch.randn(8, 16, 2, 192, device="cuda", dtype=torch.float16)
v, table, n = torch.randn_like(k), torch.arange(8, device="cuda", dtype=torch.int32).view(1, 8), torch.tensor([100], device="cuda", dtype=torch.int32)
q, mass = torch.randn(1, 1, 4, 192, device="cuda", dtype=torch.float16), torch.zeros(8, 2, 16, device="cuda")
x = torch.randn(1, 1, 2, 64, device="cuda", dtype=torch.float16)
fa2.rotary_axes_func(x, None, torch.ones(1, 1, 1, device="cuda", dtype=torch.int32), torch.rand(32, device="cuda"), (32,))  # some call
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, lse = fa2.paged_fwd(q, k, v, table, n, attn_mass=mass)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, fa2.paged_fwd(q, k, v, table, n)[0])
print("done")
"""


def test_a_kernel_whose_first_call_is_captured():
    run = subprocess.run([sys.executable, "-c", CAPTURE], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "done" in run.stdout, run.stdout + run.stderr[-2000:]


def test_masked_places_may_hold_anything():
    """Infinities and NaN where some rows of a call see a key and others do not: only the rows that see it get them."""
    import flash_attn2_b200 as fa2

    lengths, sq, h, hk, d, page = [100, 18], 3, 4, 2, 128, 16
    for bad in (math.inf, -math.inf, math.nan):
        k, v, table = make_cache(4, lengths, hk, d, page, torch.bfloat16)
        clean = v.clone()
        q = torch.randn(2, sq, h, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
        for b, n in enumerate(lengths):
            v[table[b, (n - 1) // page], (n - 1) % page, 0, 5] = bad       # seen by the last row alone
            v[table[b, (n - 14) // page], (n - 14) % page, 1, 70] = bad    # with the window by the first rows alone
        for window in (-1, 11):
            out, lse = fa2.paged_fwd(q, k, v, table, _table(lengths), window_size_left=window)
            ref, ref_lse = fa2.paged_fwd(q, k, clean, table, _table(lengths), window_size_left=window)
            assert torch.equal(lse, ref_lse)
            # the path for such values sums in another order: a rounding more or less
            differ = ~torch.isclose(out, ref, rtol=2 ** -7, atol=1e-5).cpu()
            expected = torch.zeros_like(differ)
            expected[:, 2, :2, 5] = True
            # row i stands at n - 3 + i and sees from n - 14 + i on
            expected[:, :1 if window >= 0 else 3, 2:, 70] = True
            assert torch.equal(differ, expected)
            assert not out[expected.cuda()].isfinite().any()


def test_scores_that_are_not_numbers_stay_in_their_rows():
    import flash_attn2_b200 as fa2

    lengths = [40, 200]
    k, v, table = make_cache(6, lengths, 2, 64, 16, torch.float16)
    q = torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(5)).half().cuda()
    want = fa2.paged_fwd(q, k, v, table, _table(lengths))
    q[0, 0, 1, 3] = math.nan
    got = fa2.paged_fwd(q, k, v, table, _table(lengths))
    assert got[0][0, 0, 1].isnan().all() and got[1][0, 1].isnan().all()
    keep = torch.ones(2, 1, 4, dtype=torch.bool)
    keep[0, 0, 1] = False
    assert torch.equal(got[0][keep.cuda()], want[0][keep.cuda()]) and fa2.cabi_ops.device_status() == 0


def test_views_of_q_and_out():
    import flash_attn2_b200 as fa2

    lengths, h, hk, d = [70, 333], 8, 2, 96
    k, v, table = make_cache(7, lengths, hk, d, 32, torch.bfloat16)
    q = torch.randn(2, 2, h, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    want, lse = fa2.paged_fwd(q, k, v, table, _table(lengths))
    wide = torch.nn.functional.pad(table, (3, 5), value=-7)[:, 3:-5]           # a wider table's columns
    odd = torch.nn.functional.pad(q, (0, 1))[..., :d]
    heads = q.transpose(1, 2).contiguous().transpose(1, 2)
    for x in (odd, heads, q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(fa2.paged_fwd(x, k, v, wide, _table(lengths))[0], want)
    buffers = [torch.empty_like(q), torch.full((2, 2, h, d + 8), 9.0).bfloat16().cuda()[..., :d], torch.empty(2, 2, h, d + 1).bfloat16().cuda()[..., 1:],
               torch.empty(2, h, 2, d).bfloat16().cuda().transpose(1, 2)]
    for out in buffers:
        got = fa2.paged_fwd(q, k, v, table, _table(lengths), out=out)
        assert got[0] is out and torch.equal(out, want) and torch.equal(got[1], lse)
    wide_out = torch.full((2, 4, h + 2, d + 8), 9.0).bfloat16().cuda()      # nothing is written around the output
    fa2.paged_fwd(q, k, v, table, _table(lengths), out=wide_out[:, 1:3, 1:-1, :d])
    assert torch.equal(wide_out[:, 1:3, 1:-1, :d], want)
    wide_out[:, 1:3, 1:-1, :d] = 9.0
    assert (wide_out == 9.0).all()
    same = q.clone()
    assert torch.equal(fa2.paged_fwd(same, k, v, table, _table(lengths), out=same)[0], want)


def test_pages_that_sequences_share():
    """Weights of a page in two tables add up."""
    import flash_attn2_b200 as fa2

    k, v, table = make_cache(8, [64, 64], 2, 64, 16, torch.float16)
    table[1, :2] = table[0, :2]
    lengths, q = [64, 50], torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(5)).half().cuda()
    mass = torch.zeros(k.shape[0], 2, 16, device="cuda")
    out, lse = fa2.paged_fwd(q, k, v, table, _table(lengths), attn_mass=mass)
    want = attend(q, k, v, table, lengths)
    _close(out, lse, want, torch.float16, v, 64)
    both = want[2][0][:, :32] + want[2][1][:, :32]
    torch.testing.assert_close(mass[table[0, :2].long()].cpu().double().transpose(0, 1).flatten(1), both, rtol=2 ** -22, atol=4 * want[3])


def test_pages_and_lengths_that_cannot_be():
    """A page outside the pool is seen by nobody, a length past the table is cut; both are told by the status."""
    import flash_attn2_b200 as fa2

    lengths = [64, 40]
    k, v, table = make_cache(9, lengths, 2, 64, 16, torch.bfloat16)
    q = torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        broken = table.clone()
        broken[0, 3] = bad
        mass = torch.zeros(k.shape[0], 2, 16, device="cuda")
        out, lse = fa2.paged_fwd(q, k, v, broken, _table(lengths), attn_mass=mass)
        assert fa2.cabi_ops.device_status() == 100
        want = fa2.paged_fwd(q, k, v, table, _table([48, 40]))
        _close(out, lse, (want[0].cpu().double(), want[1].cpu().double(), None, 1e-5), torch.bfloat16, v, 64)
        assert abs(mass.sum().item() - 8) < 1e-4
    want = fa2.paged_fwd(q, k, v, table, _table(lengths))
    got = fa2.paged_fwd(q, k, v, table, _table([2 ** 31 - 1, 40]))
    assert fa2.cabi_ops.device_status() == 101 and torch.equal(got[0], want[0])
    got = fa2.paged_fwd(q, k, v, table, _table(lengths), max_seqlen_k=41)
    assert fa2.cabi_ops.device_status() == 101
    assert torch.equal(got[0], fa2.paged_fwd(q, k, v, table, _table([41, 40]), max_seqlen_k=41)[0])
    got = fa2.paged_fwd(q, k, v, table, _table([-5, 40]))
    assert fa2.cabi_ops.device_status() == 0 and not got[0][0].any() and got[1][0].isinf().all()


def test_workspace_contents_do_not_matter():
    """One buffer for calls of several shapes, filled with anything, through the C entry point."""
    from flash_attn2_b200 import _cabi

    lib = _cabi.load()
    buf = torch.zeros(32 << 20, dtype=torch.uint8, device="cuda")
    keep = []

    def call(lengths, h, hk, d, fill):
        k, v, table = make_cache(10, lengths, hk, d, 16, torch.bfloat16)
        q = torch.randn(len(lengths), 1, h, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
        out, lse, n = torch.empty_like(q), torch.empty(len(lengths), h, 1, device="cuda"), _table(lengths)
        c = _cabi.PagedCache(size=C.sizeof(_cabi.PagedCache), k=k.data_ptr(), v=v.data_ptr(), k_stride=k.stride()[:3], v_stride=v.stride()[:3],
                             block_table=table.data_ptr(), block_table_stride=table.stride(0), seqlens_k=n.data_ptr(), num_pages=k.shape[0],
                             page_size=16, max_pages=table.shape[1], batch=len(lengths), heads_k=hk, head_dim=d, dtype=_cabi.FA2_BF16)
        a = _cabi.PagedFwdArgs(size=C.sizeof(_cabi.PagedFwdArgs), cache=C.pointer(c), q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
                               q_stride=q.stride()[:3], o_stride=out.stride()[:3], seqlen_q=1, heads=h, softmax_scale=d ** -0.5, window_left=-1)
        need = lib.fa2_paged_fwd_workspace_bytes(C.byref(a))
        assert 0 < need <= buf.numel()
        fill(need)
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.fa2_paged_fwd(C.byref(a), buf.data_ptr(), need - 1, stream) == -1
        assert lib.fa2_paged_fwd(C.byref(a), buf.data_ptr() + 16, need, stream) == -1
        _cabi.check(lib.fa2_paged_fwd(C.byref(a), buf.data_ptr(), need, stream))
        torch.cuda.synchronize()
        keep.append((k, v, q, table, n))
        return out, lse

    shapes = [([5000], 8, 2, 128), ([300, 2000, 5], 16, 4, 64), ([3000], 8, 2, 128), ([1500, 100], 4, 4, 256)]
    want = [call(*s, lambda n: buf.zero_()) for s in shapes]
    for fill in (lambda n: None, lambda n: buf.fill_(0xFF), lambda n: buf[:n].random_(0, 256), lambda n: buf.fill_(1)):
        for s, (out, lse) in zip(shapes, want):
            o, l = call(*s, fill)
            assert torch.equal(o, out) and torch.equal(l, lse)


def test_graphs_that_share_a_pool_and_lengths_that_grow():
    """Two captured steps over one memory pool, replayed in turns with other lengths."""
    import flash_attn2_b200 as fa2

    lengths = [900, 3000]
    k, v, table = make_cache(11, lengths, 2, 128, 16, torch.bfloat16)
    q = torch.randn(2, 1, 16, 128, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    n, mass = _table(lengths), torch.zeros(k.shape[0], 2, 16, device="cuda")
    fa2.paged_fwd(q, k, v, table, n, attn_mass=mass)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    pool = None
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool, stream=side):
            outs.append(fa2.paged_fwd(q, k, v, table, n, attn_mass=mass))
        pool = graph.pool()
        graphs.append(graph)
    for step in range(6):
        now = [900 - 100 * step, 3000 - 37 * step]
        n.copy_(_table(now))
        mass.zero_()
        graphs[step % 2].replay()
        got = [t.clone() for t in outs[step % 2]] + [mass.clone()]
        mass.zero_()
        want = [*fa2.paged_fwd(q, k, v, table, n, attn_mass=mass), mass]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert fa2.cabi_ops.device_status() == 0


def test_two_streams_at_once():
    import flash_attn2_b200 as fa2

    lengths = [2000, 1111, 600]
    k, v, table = make_cache(12, lengths, 2, 128, 16, torch.float16)
    q = torch.randn(3, 1, 8, 128, generator=torch.Generator().manual_seed(5)).half().cuda()
    n = _table(lengths)
    want = fa2.paged_fwd(q, k, v, table, n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append(fa2.paged_fwd(q, k, v, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(g[0], want[0]) and torch.equal(g[1], want[1]) for g in got)


def test_offsets_past_32_bits():
    """A pool of 2^31 elements and more; the sequence's pages are its last ones."""
    import flash_attn2_b200 as fa2

    hk, d, page = 8, 128, 64
    pages = 2 ** 31 // (hk * d * page) + 40
    k = torch.zeros(pages, page, hk, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    small_k, small_v, table = make_cache(13, [1000], hk, d, page, torch.bfloat16, spare=0)
    k[-16:], v[-16:] = small_k, small_v
    q = torch.randn(1, 1, 32, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    n = _table([1000])
    mass, small_mass = torch.zeros(pages, hk, page, device="cuda"), torch.rand(16, hk, page, device="cuda")
    mass[-16:] = small_mass
    high = (table + (pages - 16)).int()
    want = fa2.paged_fwd(q, small_k, small_v, table, n, attn_mass=small_mass)
    got = fa2.paged_fwd(q, k, v, high, n, attn_mass=mass)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(mass[-16:], small_mass)
    # append one token and evict down to 100, from the pool's end to its other half
    new = torch.randn(1, 1, hk, d, device="cuda").bfloat16()
    pos, freq = torch.full((1, 1, 1), 1000, device="cuda"), torch.rand(64, device="cuda")
    fa2.paged_append(None, new, new, k, v, high, n, pos, freq, (64,))
    assert torch.equal(v[high[0, 15].long(), 1000 - 15 * 64], new[0, 0])
    dst = torch.arange(2, device="cuda", dtype=torch.int32)[None] + (pages - 20)
    lengths, kept = fa2.paged_evict(k, v, mass, high, _table([1001]), dst, 100, 5)
    assert lengths.tolist() == [100]
    for head in range(hk):
        i = kept[0, head].long()
        j = torch.arange(100, device="cuda")
        assert torch.equal(k[dst[0].long()[j // page], j % page, head], k[high[0].long()[i // page], i % page, head])
        assert torch.equal(mass[dst[0].long()[j // page], head, j % page], mass[high[0].long()[i // page], head, i % page])
    assert fa2.cabi_ops.device_status() == 0


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("case", [
    # lengths before, new tokens of each, h, hk, d, page, sections, interleaved_axes, interleaved_pairs
    ([0], [1], 4, 2, 64, 16, (32,), False, False),
    ([15, 16, 17], [1, 1, 1], 32, 8, 128, 16, (16, 24, 24), False, False),
    ([0, 5, 100], [40, 3, 0], 8, 2, 128, 16, (24, 20, 20), True, False),     # ragged: padded rows
    ([63, 7], [130, 129], 4, 4, 96, 48, (8, 12, 12), False, True),
    ([3, 2], [9, 4], 3, 1, 72, 7, (3, 4, 5, 8), False, False),               # two bytes at a time
    ([1, 0, 2], [7, 8, 1], 4, 2, 256, 5, (128,), False, True),
], ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("form", ["dense", "packed"])
def test_append(case, dtype, form):
    import flash_attn2_b200 as fa2

    before, new, h, hk, d, page, sections, ia, ip = case
    b, s = len(before), max(new)
    k, v, table = make_cache(20, [x + y for x, y in zip(before, new)], hk, d, page, dtype, layout="hnd" if b == 3 else "nhd")
    g = torch.Generator().manual_seed(21)
    q, kn, vn = (torch.randn(b, s, n, d, generator=g).to(dtype) for n in (h, hk, hk))
    positions = torch.randint(0, 100000, (len(sections), b, s), generator=g)
    freq = torch.rand(sum(sections), generator=g)
    want_k, want_v = k.clone(), v.clone()
    turned = turn(kn, positions, freq, sections, ia, ip)
    versions = k._version, v._version
    rest = (freq.cuda(), sections, ia, ip)
    if form == "dense":
        fresh = None if len(set(new)) == 1 else _table(new)
        out = fa2.paged_append(q.cuda(), kn.cuda(), vn.cuda(), k, v, table, _table(before), positions.cuda(), *rest, seqlens_new=fresh)
        torch.testing.assert_close(out.cpu().double(), turn(q, positions, freq, sections, ia, ip), **turn_tolerance(q, dtype))
    else:
        pack = lambda t: torch.cat([t[i, :n] for i, n in enumerate(new)] + [t[0, :1]]).cuda()  # noqa: E731  (a row behind the last sequence)
        pos = torch.cat([positions[:, i, :n] for i, n in enumerate(new)] + [positions[:, 0, :1]], 1).cuda()
        cu = _table([sum(new[:i]) for i in range(b + 1)])
        out = fa2.paged_append(pack(q), pack(kn), pack(vn), k, v, table, _table(before), pos, *rest, cu_seqlens=cu)
        torch.testing.assert_close(out.cpu().double(), pack(turn(q, positions, freq, sections, ia, ip)).cpu(), **turn_tolerance(q, dtype))
    assert fa2.cabi_ops.device_status() == 0
    assert (k._version, v._version) == (versions[0] + 1, versions[1] + 1)
    rounded = torch.zeros(k.shape[:2], dtype=torch.bool)
    for i, n in enumerate(new):
        slot = torch.arange(before[i], before[i] + n)
        at = table[i].long().cpu()[slot // page], slot % page
        torch.testing.assert_close(k.cpu()[at].double(), turned[i, :n], **turn_tolerance(kn, dtype))
        assert torch.equal(v.cpu()[at], vn[i, :n])
        rounded[at] = True
    rest = ~rounded.cuda()                                    # every other row of the pool is as it was
    for now, was in ((k, want_k), (v, want_v)):
        assert torch.equal(now[rest].view(torch.int16), was[rest].view(torch.int16))


def test_append_without_a_place():
    """Tokens past the table's row, or whose page is none, go nowhere."""
    import flash_attn2_b200 as fa2

    k, v, table = make_cache(22, [40, 40], 2, 64, 16, torch.bfloat16)
    q = torch.randn(2, 1, 2, 64, device="cuda").bfloat16()
    pos, freq = torch.ones(1, 2, 1, dtype=torch.int32, device="cuda"), torch.rand(32, device="cuda")
    was = k.clone(), v.clone()
    for lengths in ([48, 2 ** 31 - 1], [-1, 48]):
        fa2.paged_append(q, q, q, k, v, table, _table(lengths), pos, freq, (32,))
        assert fa2.cabi_ops.device_status() == 100
    broken = table.clone()
    broken[:, 2] = _table([-3, k.shape[0]])
    fa2.paged_append(q, q, q, k, v, broken, _table([40, 40]), pos, freq, (32,))
    assert fa2.cabi_ops.device_status() == 100
    for now, before in ((k, was[0]), (v, was[1])):
        assert torch.equal(now.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("before,new,h,hk,d,page,sections", [
    ([15, 16, 17], [1, 1, 1], 32, 8, 128, 16, (16, 24, 24)),     # few tokens: several warps have a token
    ([0, 5, 100], [700, 3, 0], 8, 2, 128, 16, (24, 20, 20)),
    ([3, 2], [9, 4], 40, 40, 72, 7, (3, 4, 5, 8)),               # two bytes at a time, more heads than lanes
    ([0, 63], [2000, 1999], 2, 1, 64, 48, (32,)),
], ids=str)
@pytest.mark.parametrize("form", ["dense", "packed"])
def test_append_starts_the_weights(before, new, h, hk, d, page, sections, form):
    """Entries of the new tokens are 0 whatever lay there, all others the bits that they were; keys and values as without weights."""
    import flash_attn2_b200 as fa2

    b, s = len(before), max(new)
    k, v, table = make_cache(23, [x + y for x, y in zip(before, new)], hk, d, page, torch.bfloat16)
    g = torch.Generator().manual_seed(24)
    q, kn, vn = (torch.randn(b, s, n, d, generator=g).bfloat16().cuda() for n in (h, hk, hk))
    positions, freq = torch.randint(0, 1000, (len(sections), b, s), generator=g).cuda(), torch.rand(sum(sections), generator=g).cuda()
    mass = torch.randn(k.shape[0], hk, page, generator=g).cuda()
    mass[mass > 1] = math.nan
    want, other = mass.clone(), (k.clone(), v.clone())
    for i, n in enumerate(new):
        slot = torch.arange(before[i], before[i] + n, device="cuda")
        want[table[i].long()[slot // page], :, slot % page] = 0.0
    extra = dict(seqlens_new=_table(new))
    if form == "packed":
        q, kn, vn = (torch.cat([t[i, :n] for i, n in enumerate(new)] + [t[0, :1]]) for t in (q, kn, vn))
        positions = torch.cat([positions[:, i, :n] for i, n in enumerate(new)] + [positions[:, 0, :1]], 1)
        extra = dict(cu_seqlens=_table([sum(new[:i]) for i in range(b + 1)]))
    version = mass._version
    out = fa2.paged_append(q, kn, vn, k, v, table, _table(before), positions, freq, sections, attn_mass=mass, **extra)
    assert mass._version == version + 1
    assert torch.equal(fa2.paged_append(q, kn, vn, *other, table, _table(before), positions, freq, sections, **extra), out)
    for x, y in zip((k, v), other):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    assert torch.equal(mass.view(torch.int32), want.view(torch.int32))
    was = mass.clone()                                           # tokens without a place have no entries
    fa2.paged_append(q, kn, vn, k, v, table, _table([2 ** 31 - 1] * b), positions, freq, sections, attn_mass=mass, **extra)
    assert fa2.cabi_ops.device_status() == 100 and torch.equal(mass.view(torch.int32), was.view(torch.int32))


@pytest.mark.parametrize("d,sections", [(128, (64,)), (72, (20,))])
def test_tokens_that_lie_in_the_cache(d, sections):
    """Rows of the cache itself are appended, one place further on and over each other: all are read before any is written."""
    import flash_attn2_b200 as fa2

    n, page = 3000, 3100
    k, v, table = make_cache(26, [page], 2, d, page, torch.bfloat16)
    home = table[0, 0].item()
    was = k.clone(), v.clone()
    pos, freq = torch.zeros(1, 1, n, dtype=torch.int32, device="cuda"), torch.rand(sum(sections), device="cuda")
    q = fa2.paged_append(k[home:home + 1, :n], k[home:home + 1, :n], v[home:home + 1, :n], k, v, table, _table([1]), pos, freq, sections)
    assert fa2.cabi_ops.device_status() == 0 and torch.equal(q[0], was[0][home, :n])
    for now, before in ((k, was[0]), (v, was[1])):               # at position 0 a key stays what it is
        assert torch.equal(now[home, 1:n + 1], before[home, :n])
        assert torch.equal(now[home, n + 1:], before[home, n + 1:]) and torch.equal(now[home, 0], before[home, 0])


def test_append_refuses_tokens_without_memory():
    """A sparse tensor, or one on the CPU, is refused before anything asks where it lies."""
    import flash_attn2_b200 as fa2

    k, v, table = make_cache(27, [4], 2, 64, 16, torch.bfloat16)
    new, pos, freq = torch.zeros(1, 1, 2, 64, device="cuda").bfloat16(), torch.ones(1, 1, 1, dtype=torch.int32, device="cuda"), torch.rand(32, device="cuda")
    for kind, bad in ((ValueError, new.to_sparse()), (NotImplementedError, new.cpu())):
        for i in range(3):
            tokens = [new] * 3
            tokens[i] = bad
            with pytest.raises(kind):
                fa2.paged_append(*tokens, k, v, table, _table([4]), pos, freq, (32,))


def test_append_refuses_weights_of_another_form():
    import flash_attn2_b200 as fa2

    k, v, table = make_cache(25, [40, 7], 2, 64, 16, torch.bfloat16)
    new, n = torch.randn(2, 1, 2, 64, device="cuda").bfloat16(), _table([40, 7])
    pos, freq, mass = torch.ones(1, 2, 1, dtype=torch.int32, device="cuda"), torch.rand(32, device="cuda"), torch.zeros(k.shape[0], 2, 16, device="cuda")
    for kind, bad in ((ValueError, mass.transpose(1, 2)), (ValueError, mass[1:]), (TypeError, mass.double()), (NotImplementedError, mass.cpu()),
                      (TypeError, 0.0), (RuntimeError, mass.clone().requires_grad_())):
        was = k.clone()
        with pytest.raises(kind):
            fa2.paged_append(new, new, new, k, v, table, n, pos, freq, (32,), attn_mass=bad)
        assert torch.equal(k.view(torch.int16), was.view(torch.int16))


# ---------------------------------------------------------------- eviction
def _masses(seed, pages, hk, page, kind):
    g = torch.Generator().manual_seed(seed)
    m = torch.randn(pages, hk, page, generator=g)
    if kind == "heavy":
        m = torch.where(m < -0.3, torch.zeros(()), torch.exp(3 * m))
    elif kind == "ties":
        m = (m * 2).round().abs()
    elif kind == "equal":
        m = torch.full_like(m, 0.25)
    elif kind == "zeroes":
        m = torch.where(m < 0, -torch.zeros(()), torch.zeros(()))
    elif kind == "anything":                                  # negative, infinite, NaN, both zeroes
        special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1e-42, 3e38])
        m = torch.where(torch.rand(m.shape, generator=g) < 0.3, special[torch.randint(0, 8, m.shape, generator=g)], m)
    return m


@pytest.mark.parametrize("lengths,budget,recent,hk,d,page", [
    ([1], 1, 0, 1, 8, 1),
    ([5, 0, 9], 4, 1, 2, 64, 3),
    ([100, 64, 65, 63], 64, 16, 2, 128, 16),
    ([1000, 3000], 700, 700, 2, 64, 48),                     # the newest alone
    ([2500, 33], 999, 0, 3, 96, 7),
    ([4096, 5000], 2048, 100, 2, 128, 64),
    ([4097], 4096, 3, 1, 256, 100),
    ([9000], 1, 0, 2, 64, 256),
], ids=str)
@pytest.mark.parametrize("kind", ["heavy", "ties", "equal", "zeroes", "anything"])
def test_evict(lengths, budget, recent, hk, d, page, kind):
    import flash_attn2_b200 as fa2

    _evict(fa2, lengths, budget, recent, hk, d, page, kind)


def _evict(fa2, lengths, budget, recent, hk, d, page, kind):
    kept_counts = [min(n, budget) for n in lengths]
    need = [-(-n // page) for n in kept_counts]
    k, v, table = make_cache(30, lengths, hk, d, page, torch.float16, spare=0)
    first = k.shape[0]
    k, v = (torch.cat([t, torch.full((sum(need) + 1, *t.shape[1:]), 7.0, dtype=t.dtype, device="cuda")]) for t in (k, v))
    dst = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32)
    order = (torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)) + first).tolist()
    for b, n in enumerate(need):
        dst[b, :n] = torch.tensor([order.pop() for _ in range(n)])
    mass = _masses(31, k.shape[0], hk, page, kind).cuda()
    was = [t.clone() for t in (k, v, mass)]
    versions = [t._version for t in (k, v, mass)]
    got_lengths, kept = fa2.paged_evict(k, v, mass, table, _table(lengths), dst.cuda(), budget, recent=recent)
    assert fa2.cabi_ops.device_status() == 0
    assert got_lengths.tolist() == kept_counts and got_lengths.dtype == kept.dtype == torch.int32
    assert [t._version for t in (k, v, mass)] == [x + 1 for x in versions]
    want = [t.cpu().clone() for t in was]
    for b, n in enumerate(lengths):
        t = torch.arange(n)
        pages = table.cpu()[b].long()[t // page]
        for head in range(hk):
            keep = choose(was[2].cpu()[pages, head, t % page], n, budget, recent)
            assert kept[b, head].tolist() == keep + [-1] * (budget - len(keep)), (b, head)
            i, j = torch.tensor(keep, dtype=torch.long), torch.arange(len(keep))
            to, out = dst[b].long()[j // page], table.cpu()[b].long()[i // page]
            for x, y in zip(want[:2], was[:2]):
                x[to, j % page, head] = y.cpu()[out, i % page, head]
            want[2][to, head, j % page] = was[2].cpu()[out, head, i % page]
    for now, w, word in zip((k, v, mass), want, (torch.int16, torch.int16, torch.int32)):  # NaN and unused rows too, to the bit
        assert torch.equal(now.cpu().view(word), w.view(word))


@pytest.mark.parametrize("lengths", [[60000, 49153, 100], [12000], [30000, 16385, 7], [140001]], ids=str)
def test_evict_of_long_sequences(lengths):
    """Clusters of 2, 4 and 8 CTAs, and more keys than their registers hold."""
    import flash_attn2_b200 as fa2

    for kind in ("heavy", "ties"):
        _evict(fa2, lengths, max(lengths) // 3, 300, 1, 8, 128 if kind == "ties" else 50, kind)


def test_evict_of_many_long_sequences():
    """More units than SMs: a CTA each, and more keys than its registers hold. (All rows go to one page: only the choice is looked at.)"""
    import flash_attn2_b200 as fa2

    b, n, page, budget = 150, 20000, 16, 5000
    k = torch.zeros(n // page + 1, page, 1, 8, dtype=torch.float16, device="cuda")
    mass = torch.randn(k.shape[0], 1, page, device="cuda").abs().round(decimals=2)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(b, -1)
    lengths = torch.arange(n - b, n, device="cuda", dtype=torch.int32)
    want = [mass[:-1].flatten()[: m - 10].sort(descending=True, stable=True).indices[: budget - 10].sort().values for m in lengths.tolist()]
    got, kept = fa2.paged_evict(k, k.clone(), mass.clone(), table, lengths, torch.full((b, budget // page + 1), n // page, dtype=torch.int32, device="cuda"),
                                budget, recent=10)
    assert fa2.cabi_ops.device_status() == 0 and (got == budget).all()
    for i, w in enumerate(want):
        assert torch.equal(kept[i, 0, : budget - 10].long(), w) and kept[i, 0, -1] == lengths[i] - 1


def test_evict_with_pages_that_cannot_be():
    """Rows of such a page are the first to go, and move nowhere; a place that there is no page for stays empty."""
    import flash_attn2_b200 as fa2

    k, v, table = make_cache(32, [64], 1, 64, 16, torch.float16, spare=4)
    used = set(table.flatten().tolist())
    free = torch.tensor([[p for p in range(k.shape[0]) if p not in used][:2]], dtype=torch.int32).cuda()
    mass = torch.rand(k.shape[0], 1, 16, device="cuda") + 0.1
    broken = table.clone()
    broken[0, 1] = -1
    lengths, kept = fa2.paged_evict(k, v, mass, broken, _table([64]), free, 32)
    assert fa2.cabi_ops.device_status() == 100 and not set(kept.flatten().tolist()) & set(range(16, 32))
    was = k.clone()
    fa2.paged_evict(k, v, mass, table, _table([64]), free[:, :1].contiguous(), 32)      # room for 16 of 32
    assert fa2.cabi_ops.device_status() == 100
    others = [p for p in range(k.shape[0]) if p != free[0, 0].item()]
    assert torch.equal(k[others].view(torch.int16), was[others].view(torch.int16))
    lengths, kept = fa2.paged_evict(k, v, mass, table, _table([2 ** 31 - 1]), free, 32)
    assert fa2.cabi_ops.device_status() == 101 and lengths.tolist() == [32]


def test_refusals():
    import flash_attn2_b200 as fa2

    k, v, table = make_cache(33, [40, 7], 2, 64, 16, torch.bfloat16)
    n, q = _table([40, 7]), torch.randn(2, 1, 4, 64, device="cuda").bfloat16()
    mass = torch.zeros(k.shape[0], 2, 16, device="cuda")
    pos, freq, new = torch.ones(1, 2, 1, dtype=torch.int32, device="cuda"), torch.rand(32, device="cuda"), q[:, :, :2]
    cache = dict(k_cache=k, v_cache=v, block_table=table, seqlens_k=n)
    calls = {"fwd": (fa2.paged_fwd, dict(q=q)), "append": (fa2.paged_append, dict(q=q, k=new, v=new, positions=pos, inv_freq=freq, sections=(32,))),
             "evict": (fa2.paged_evict, dict(attn_mass=mass, dst_block_table=table, budget=4))}

    def refused(which, kind, **kw):
        f, args = calls[which]
        with pytest.raises(kind):
            f(**{**cache, **args, **kw})

    for which in calls:
        refused(which, ValueError, v_cache=v[1:])
        refused(which, TypeError, v_cache=v.half())
        refused(which, TypeError, k_cache=k.float(), v_cache=v.float())
        refused(which, ValueError, k_cache=k[0], v_cache=v[0])
        refused(which, ValueError, k_cache=k[..., :60], v_cache=v[..., :60])
        refused(which, ValueError, k_cache=k.transpose(2, 3), v_cache=v.transpose(2, 3))
        refused(which, ValueError, k_cache=torch.nn.functional.pad(k, (0, 1))[..., :64])
        refused(which, TypeError, block_table=table.long())
        refused(which, ValueError, block_table=table[0])
        refused(which, ValueError, block_table=table[:, :0])
        refused(which, TypeError, seqlens_k=n.long())
        refused(which, ValueError, seqlens_k=n[:1])
        refused(which, NotImplementedError, seqlens_k=n.cpu())
        refused(which, NotImplementedError, block_table=table.cpu())
        refused(which, RuntimeError, k_cache=k.clone().requires_grad_())
    refused("fwd", TypeError, q=q.half())
    refused("fwd", ValueError, q=q[:1])
    refused("fwd", ValueError, q=q[:, 0])
    refused("fwd", ValueError, q=q[..., :32])
    refused("fwd", ValueError, q=q[:, :, :3])
    refused("fwd", ValueError, q=q.expand(2, 1, 4, 64).repeat(1, 65, 1, 1))
    refused("fwd", ValueError, out=q[:, :, :2])
    refused("fwd", ValueError, out=q[:, :, :1].expand(2, 1, 4, 64))
    refused("fwd", ValueError, attn_mass=mass.transpose(1, 2))
    refused("fwd", TypeError, attn_mass=mass.double())
    refused("fwd", ValueError, softmax_scale=math.inf)
    refused("fwd", ValueError, softcap=-1.0)
    refused("fwd", ValueError, max_seqlen_k=0)
    refused("fwd", ValueError, window_size_left=2 ** 40)
    refused("fwd", TypeError, window_size_left=1.5)
    refused("fwd", RuntimeError, q=q.clone().requires_grad_())
    refused("append", ValueError, v=new[:1])
    refused("append", TypeError, v=new.half())
    refused("append", ValueError, k=q, v=q)
    refused("append", ValueError, q=None, k=new[:1], v=new[:1], positions=pos[:, :1])
    refused("append", ValueError, cu_seqlens=_table([0, 1, 2]))
    refused("append", ValueError, q=q[:, 0], k=new[:, 0], v=new[:, 0], positions=pos[:, :, 0])
    refused("append", ValueError, seqlens_new=n[:1])
    refused("append", ValueError, k_cache=k[:, :, :1].expand(-1, -1, 2, -1))
    refused("append", RuntimeError, q=q.clone().requires_grad_())
    refused("evict", TypeError, attn_mass=None)
    refused("evict", ValueError, budget=0)
    refused("evict", ValueError, recent=5)
    refused("evict", ValueError, dst_block_table=table[:1])
    refused("evict", TypeError, dst_block_table=table.long())
    assert fa2.cabi_ops.device_status() == 0


def test_empty_batches():
    import flash_attn2_b200 as fa2

    k, v, table = make_cache(34, [40], 2, 64, 16, torch.bfloat16)
    none, nobody = table[:0], _table([])
    out, lse = fa2.paged_fwd(torch.empty(0, 1, 4, 64, device="cuda").bfloat16(), k, v, none, nobody)
    assert out.shape == (0, 1, 4, 64) and lse.shape == (0, 4, 1)
    out, lse = fa2.paged_fwd(torch.empty(1, 0, 4, 64, device="cuda").bfloat16(), k, v, table, _table([40]))
    assert out.shape == (1, 0, 4, 64) and lse.shape == (1, 4, 0)
    lengths, kept = fa2.paged_evict(k, v, torch.zeros(k.shape[0], 2, 16, device="cuda"), none, nobody, none, 4)
    assert lengths.shape == (0,) and kept.shape == (0, 2, 4)
    q = torch.empty(1, 0, 2, 64, device="cuda").bfloat16()
    assert fa2.paged_append(q, q, q, k, v, table, _table([40]), torch.empty(1, 1, 0, dtype=torch.int32, device="cuda"), torch.rand(32, device="cuda"),
                            (32,)).shape == q.shape


def test_a_run_as_it_would_be_used():
    """A prompt is appended, tokens are decoded with account of their weights, each head drops what got least, and decoding goes on:
    every step against dense attention in 64 bits over what each head still has."""
    import flash_attn2_b200 as fa2

    b, h, hk, d, page, sections = 2, 8, 2, 64, 16, (12, 10, 10)
    prompts, budget, recent = [150, 90], 64, 16
    g = torch.Generator().manual_seed(40)
    freq = 1e4 ** (-torch.arange(32, dtype=torch.float32) / 32)
    k = torch.full((60, page, hk, d), math.nan, dtype=torch.bfloat16, device="cuda")
    v, mass = k.clone(), torch.zeros(60, hk, page, device="cuda")
    table = torch.randperm(60, generator=g)[:24].view(2, 12).int().cuda()
    spare = torch.tensor([sorted(set(range(60)) - set(table.flatten().tolist()))[:12]]).view(2, 6).int().cuda()
    n = _table([0, 0])
    have = [[[] for _ in range(hk)] for _ in range(b)]         # (key, value) rows of each head, in the cache's order
    heads = []

    def append(count):
        s = max(count)
        q, kn, vn = (torch.randn(b, s, x, d, generator=g).bfloat16() for x in (h, hk, hk))
        at = torch.arange(s) + torch.tensor([len(have[i][0]) for i in range(b)])[:, None]
        pos = torch.stack([at, at // 5, at % 5])
        out = fa2.paged_append(q.cuda(), kn.cuda(), vn.cuda(), k, v, table, n, pos.cuda(), freq.cuda(), sections, seqlens_new=_table(count))
        turned = fa2.rotary_axes_func(q.cuda(), kn.cuda(), pos.cuda(), freq.cuda(), sections)
        assert torch.equal(out, turned[0])                     # the same turn as in training
        for i in range(b):
            for x in range(hk):
                have[i][x] += [(turned[1][i, t, x].cpu().double(), vn[i, t, x].double()) for t in range(count[i])]
        n.add_(_table(count))
        return out

    def decode():
        q = append([1, 1])
        out, lse = fa2.paged_fwd(q, k, v, table, n, attn_mass=mass, max_seqlen_k=192)
        for i in range(b):
            for x in range(h):
                keys, values = (torch.stack(t) for t in zip(*have[i][x // (h // hk)]))
                p = torch.softmax(keys @ q[i, 0, x].cpu().double() * d ** -0.5, 0)
                torch.testing.assert_close(out[i, 0, x].cpu().double(), p @ values, rtol=2 ** -8 * 1.01, atol=1e-3)
                heads.append(p)

    append(prompts)
    for _ in range(4):
        decode()
    total = mass.sum().item()
    assert abs(total - 4 * b * h) < 1e-3
    lengths, kept = fa2.paged_evict(k, v, mass, table, n, spare, budget, recent=recent)
    for i in range(b):
        for x in range(hk):
            assert sorted(kept[i, x].tolist())[-recent:] == list(range(len(have[i][x]) - recent, len(have[i][x])))
            have[i][x] = [have[i][x][t] for t in kept[i, x].tolist() if t >= 0]
    table, n = spare, lengths
    for _ in range(4):
        decode()
    assert n.tolist() == [68, 68] and fa2.cabi_ops.device_status() == 0


@pytest.mark.parametrize("page", [16, 12])
def test_pages_that_are_used_again(page):
    """A server's life: sequences decode with account of their weights and are evicted again and again between two halves of a small pool,
    whose rows hold keys and weights of tokens that are gone. Each token's weight is the sum of what it got itself, in 64 bits, and the
    choice goes by it."""
    import flash_attn2_b200 as fa2

    b, h, hk, d, sections, budget, recent = 2, 4, 2, 64, (32,), 40, 8
    g = torch.Generator().manual_seed(41)
    freq = 1e4 ** (-torch.arange(32, dtype=torch.float32) / 32).cuda()
    room = 80 // page + 1
    k = torch.randn(4 * room, page, hk, d, generator=g).bfloat16().cuda()
    v, mass = k.clone(), torch.full((4 * room, hk, page), math.nan, device="cuda")
    pages = torch.randperm(4 * room, generator=g).int().cuda()
    halves = [pages[: 2 * room].view(2, room).contiguous(), pages[2 * room:].view(2, room).contiguous()]
    n, at = _table([0, 0]), 0
    have = [[[] for _ in range(hk)] for _ in range(b)]           # [key, weight] of each head, in the cache's order
    worst = 0.0                                                  # sums of the magnitudes of the scores' products
    for life in range(4):
        table = halves[life % 2]
        for step in range(12):
            count = [30, 17] if life == step == 0 else [3, 2] if step == 0 else [1, 1]
            s = max(count)
            q, kn, vn = (torch.randn(b, s, x, d, generator=g).bfloat16() for x in (h, hk, hk))
            pos = (at + torch.arange(s).expand(1, b, s)).cuda()
            at += s
            qt = fa2.paged_append(q.cuda(), kn.cuda(), vn.cuda(), k, v, table, n, pos, freq, sections, seqlens_new=_table(count), attn_mass=mass)
            kt = fa2.rotary_axes_func(None, kn.cuda(), pos, freq, sections)[1].cpu().double()
            n = n + _table(count)
            last = torch.stack([qt[i, c - 1: c] for i, c in enumerate(count)])
            fa2.paged_fwd(last, k, v, table, n, attn_mass=mass, max_seqlen_k=room * page)
            for i in range(b):
                for x in range(hk):
                    have[i][x] += [[kt[i, t, x], 0.0] for t in range(count[i])]
                    keys = torch.stack([e[0] for e in have[i][x]])
                    for head in range(x * (h // hk), (x + 1) * (h // hk)):
                        qr = last[i, 0, head].cpu().double()
                        worst = max(worst, (keys.abs() @ qr.abs()).max().item() * d ** -0.5)
                        p = torch.softmax(keys @ qr * d ** -0.5, 0)
                        for e, w in zip(have[i][x], p.tolist()):
                            e[1] += w
        to = halves[1 - life % 2]
        lengths, kept = fa2.paged_evict(k, v, mass, table, n, to, budget, recent=recent)
        for i in range(b):
            for x in range(hk):
                t = torch.arange(len(have[i][x]))
                got = mass.cpu()[table.cpu()[i].long()[t // page], x, t % page]
                # twice the scores' error (as in attend), exp2's 2^-22 and the roundings of up to 100 sums
                torch.testing.assert_close(got.double(), torch.tensor([e[1] for e in have[i][x]], dtype=torch.float64),
                                           rtol=2 * (d + 16) * 2.0 ** -23 * worst + 2.0 ** -22 + 100 * 2.0 ** -24, atol=0)
                keep = choose(got, len(have[i][x]), budget, recent)
                assert kept[i, x].tolist() == keep + [-1] * (budget - len(keep))
                have[i][x] = [have[i][x][j] for j in keep]
        n = lengths
    assert fa2.cabi_ops.device_status() == 0


@pytest.mark.parametrize("sink", [12.0, 16.0, 17.5, 19.0])
@pytest.mark.parametrize("h,d,page", [(1, 64, 16), (1, 128, 9), (12, 128, 16), (20, 128, 16), (20, 256, 16), (3, 192, 16)])
def test_a_key_that_has_nearly_all_the_weight(h, d, page, sink):
    """The first key's score is far above the others', whose weights (2^-17 to 2^-27) would be too small for fp16's subnormals as they
    are, while their values, all of one sign, make the output: none of them gets lost. (160 sequences on the same pages, so that a
    unit's keys lie in the warps of one or two CTAs.)"""
    import flash_attn2_b200 as fa2

    n, b, large = 2048, 160, 60000.0
    pages = -(-n // page)
    k = torch.zeros(pages, page, 1, d, dtype=torch.float16, device="cuda")
    v = torch.full_like(k, large)
    k[0, 0, 0, 0], v[0, 0] = sink, 1.0
    q = torch.zeros(b, 1, h, d, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(b, -1)
    out, lse = fa2.paged_fwd(q, k, v, table, _table([n] * b), softmax_scale=1.0)
    tail = (n - 1) * math.exp(-sink)
    want = (1.0 + tail * large) / (1.0 + tail)
    # Scores: one product, times log2 e, both roundings 2^-24 of at most 27.5; the differences' weights are off by 2^-17 of themselves. P's
    # error is at most half a step of fp16's subnormals at 2^7 of the largest weight, 2^-32 of that, for each key.
    atol = tail * large * 2.0 ** -17 + n * 2.0 ** -32 * large
    torch.testing.assert_close(out.double(), torch.full_like(out, want, dtype=torch.float64), rtol=2.0 ** -11 * 1.001, atol=atol)
    torch.testing.assert_close(lse.double(), torch.full_like(lse, sink + math.log1p(tail), dtype=torch.float64), rtol=2.0 ** -22, atol=2.0 ** -20)


@pytest.mark.parametrize("window", [-1, 70])
def test_a_chunk_of_a_prompt_in_pieces(window):
    """More rows than a call takes are refused with the way to go: pieces of the chunk, each with the lengths that end at its last token,
    are the rows of the chunk, and their weights its weights."""
    import flash_attn2_b200 as fa2

    lengths, s, h, hk, d, most = [700, 301], 301, 8, 2, 64, 32
    k, v, table = make_cache(42, lengths, hk, d, 16, torch.bfloat16)
    q = torch.randn(2, s, h, d, generator=torch.Generator().manual_seed(43)).bfloat16().cuda()
    with pytest.raises(ValueError, match="in pieces, each with lengths up to its own last token"):
        fa2.paged_fwd(q, k, v, table, _table(lengths))
    mass = torch.zeros(k.shape[0], hk, 16, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(2, h, s, device="cuda")
    for i in range(0, s, most):
        j = min(s, i + most)
        out[:, i:j], lse[:, :, i:j] = fa2.paged_fwd(q[:, i:j], k, v, table, _table(lengths) - s + j, attn_mass=mass, window_size_left=window)
    want = attend(q, k, v, table, lengths, window=window)
    assert fa2.cabi_ops.device_status() == 0
    _close(out, lse, want, torch.bfloat16, v, 700)
    for b, n in enumerate(lengths):
        got = mass[table[b].long().clamp(min=0)].transpose(1, 2).flatten(0, 1)[:n].T.cpu().double()
        # each piece's sum, and the additions of ten of them
        torch.testing.assert_close(got, want[2][b], rtol=10 * 2.0 ** -24, atol=2 * want[3] * s * (h // hk))


@pytest.mark.parametrize("d", [8, 16, 40, 56, 88, 120, 136, 168, 200, 248])
def test_head_dims_between_the_boxes(d):
    """Pages of whole tiles at head dims that leave the last box of 64 columns partly outside."""
    import flash_attn2_b200 as fa2

    lengths = [33, 400, 0]
    k, v, table = make_cache(44, lengths, 2, d, 32, torch.float16)
    q = torch.randn(3, 2, 12, d, generator=torch.Generator().manual_seed(45)).half().cuda()
    out, lse = fa2.paged_fwd(q, k, v, table, _table(lengths))
    assert fa2.cabi_ops.device_status() == 0
    _close(out, lse, attend(q, k, v, table, lengths), torch.float16, v, 400)


def test_append_of_keys_alone():
    """No queries: keys, values and weights as with them."""
    import flash_attn2_b200 as fa2

    for d, sections in ((64, (32,)), (72, (3, 4))):
        k, v, table = make_cache(46, [20, 9], 2, d, 16, torch.float16)
        new = torch.randn(2, 3, 2, d, generator=torch.Generator().manual_seed(47)).half().cuda()
        pos, freq = torch.arange(3, device="cuda").expand(len(sections), 2, 3), torch.rand(sum(sections), device="cuda")
        want, mass = (k.clone(), v.clone()), torch.ones(k.shape[0], 2, 16, device="cuda")
        mass_want = mass.clone()
        fa2.paged_append(new, new, new, *want, table, _table([17, 6]), pos, freq, sections, attn_mass=mass_want)
        assert fa2.paged_append(None, new, new, k, v, table, _table([17, 6]), pos, freq, sections, attn_mass=mass) is None
        assert fa2.cabi_ops.device_status() == 0
        for now, w in zip((k, v), want):
            assert torch.equal(now.view(torch.int16), w.view(torch.int16))
        assert torch.equal(mass, mass_want) and (mass == 0).sum() == 2 * 2 * 3
