"""GPU: rotary positions with several axes against 64-bit arithmetic: sections and turns, both kinds of pairs, heads that are turned in
part, odd numbers of pairs, strided and unaligned tensors, far positions, gradients of both orders."""
import subprocess
import sys

import pytest
import torch

from tests._paged import turn, turn_tolerance

pytestmark = pytest.mark.gpu

# b, s, h, hk, d, sections, interleaved_axes, interleaved_pairs
CASES = [
    (1, 1, 1, 1, 8, (4,), False, False),
    (1, 1, 32, 8, 128, (16, 24, 24), False, False),
    (2, 577, 16, 4, 96, (8, 12, 12), False, True),        # a third of each head is copied
    (2, 63, 12, 12, 64, (12, 10, 10), True, False),
    (3, 40, 4, 1, 256, (44, 42, 42), True, True),
    (1, 300, 5, 5, 72, (3, 4, 5, 8), False, False),        # 20 pairs: two bytes at a time
    (2, 33, 3, 1, 40, (7, 0, 2), False, True),              # 9 pairs, an axis without any
    (1, 129, 8, 2, 136, (8,), False, False),               # 8 pairs of 68
    (1, 50, 64, 8, 128, (24, 20, 20), True, False),
    (4, 1000, 2, 2, 192, (32, 32, 32), True, False),
]


def _inputs(seed, b, s, h, hk, d, sections, dtype, far=200000):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(b, s, h, d, generator=g).to(dtype), torch.randn(b, s, hk, d, generator=g).to(dtype)
    n = sum(sections)
    positions = torch.randint(0, far, (len(sections), b, s), generator=g)
    inv_freq = 1e4 ** (-torch.arange(n, dtype=torch.float32) / n)
    return q, k, positions, inv_freq


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("int64", [True, False], ids=["i64", "i32"])
def test_forward(case, dtype, int64):
    import flash_attn2_b200 as fa2

    b, s, h, hk, d, sections, ia, ip = case
    q, k, positions, inv_freq = _inputs(1, b, s, h, hk, d, sections, dtype)
    at = positions.cuda() if int64 else positions.int().cuda()
    got = fa2.rotary_axes_func(q.cuda(), k.cuda(), at, inv_freq.cuda(), sections, ia, ip)
    for g, x in zip(got, (q, k)):
        torch.testing.assert_close(g.cpu().double(), turn(x, positions, inv_freq, sections, ia, ip), **turn_tolerance(x, dtype))
        assert g.is_contiguous() and g.dtype == dtype


def test_one_of_the_two_and_packed_rows():
    import flash_attn2_b200 as fa2

    q, k, positions, inv_freq = _inputs(2, 1, 70, 6, 2, 64, (12, 10, 10), torch.bfloat16)
    qc, kc, pc, fc = (t.cuda() for t in (q, k, positions, inv_freq))
    a, b = fa2.rotary_axes_func(qc, kc, pc, fc, (12, 10, 10))
    assert fa2.rotary_axes_func(None, kc, pc, fc, [12, 10, 10])[0] is None
    assert torch.equal(fa2.rotary_axes_func(qc, None, pc, fc, (12, 10, 10))[0], a)
    assert torch.equal(fa2.rotary_axes_func(None, kc, pc, fc, (12, 10, 10))[1], b)
    c, e = fa2.rotary_axes_func(qc[0], kc[0], pc[:, 0], fc, (12, 10, 10))
    assert torch.equal(c, a[0]) and torch.equal(e, b[0])


@pytest.mark.parametrize("view", ["fused", "heads_first", "odd_offset", "odd_stride", "last", "broadcast"])
def test_layouts(view):
    """Views that the wide loads cannot take are turned two bytes at a time; the results are the same bits."""
    import flash_attn2_b200 as fa2

    b, s, h, hk, d, sections = 2, 45, 8, 8, 64, (12, 10, 10)
    q, k, positions, inv_freq = (t.cuda() for t in _inputs(3, b, s, h, hk, d, sections, torch.float16))
    if view == "broadcast":
        k = k[:, :, :1].expand(b, s, hk, d)
        positions = positions[:1, :1].expand(3, b, s)
    want = fa2.rotary_axes_func(q, k.contiguous(), positions.contiguous(), inv_freq, sections)
    if view == "fused":
        both = torch.cat([q, k], 2)
        q, k = both[:, :, :h], both[:, :, h:]
    elif view == "heads_first":
        q, k = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k))
    elif view == "odd_offset":
        q = torch.cat([q.flatten()[:1], q.flatten()])[1:].view(q.shape)
    elif view == "odd_stride":
        k = torch.nn.functional.pad(k, (0, 3))[..., :d]
    elif view == "last":
        q = q.transpose(2, 3).contiguous().transpose(2, 3)
    got = fa2.rotary_axes_func(q, k, positions, inv_freq, sections)
    if view in ("odd_offset", "odd_stride"):  # another order of the same sums: the roundings may differ
        for g, w in zip(got, want):
            torch.testing.assert_close(g, w, rtol=2 ** -10, atol=1e-6)
    else:
        assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("positions", [[0, 1, -1, 2 ** 20, -2 ** 20], [2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 2 ** 24 + 1, 7], [2 ** 33, 2 ** 35 + 3, -2 ** 34, 0, 1]])
def test_far_positions(positions):
    """Angles of 2^31 turns and more; the sine of a small angle keeps its own precision."""
    import flash_attn2_b200 as fa2

    x = torch.ones(1, 5, 1, 16, dtype=torch.float16)
    inv_freq = torch.tensor([1.0, 0.73, 3.1415927, 1e-3, 1e-9, 6.2831855, 0.0, 12.5])
    at = torch.tensor(positions).view(1, 1, 5)
    got = fa2.rotary_axes_func(x.cuda(), None, at.cuda(), inv_freq.cuda(), (8,))[0]
    # pos * f in fp64 is itself off by pos * f * 2^-53, the fixed-point fraction by as much, the rest as everywhere.
    far = max(abs(p) for p in positions) * 12.5 * 2.0 ** -52
    torch.testing.assert_close(got.cpu().double(), turn(x, at, inv_freq, (8,)), rtol=2 ** -11 * 1.001, atol=4e-6 + 2 * far)


def test_frequencies_that_are_no_numbers():
    import flash_attn2_b200 as fa2

    x = torch.ones(1, 2, 1, 16, dtype=torch.bfloat16, device="cuda")
    inv_freq = torch.full((8,), 0.5, device="cuda")
    inv_freq[2], inv_freq[5] = float("nan"), float("inf")
    got = fa2.rotary_axes_func(x, None, torch.ones(1, 1, 2, dtype=torch.int32, device="cuda"), inv_freq, (8,))[0]
    bad = got.isnan()[0, 0, 0].nonzero().flatten().tolist()
    assert bad == [2, 5, 10, 13]


@pytest.mark.parametrize("shape", [(0, 5), (2, 0)])
def test_empty(shape):
    import flash_attn2_b200 as fa2

    q = torch.empty(*shape, 4, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    k = torch.empty(*shape, 2, 64, dtype=torch.bfloat16, device="cuda")
    a, b = fa2.rotary_axes_func(q, k, torch.empty(1, *shape, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda"), (32,))
    a.sum().backward()
    assert a.shape == q.shape and b.shape == k.shape and q.grad.shape == q.shape


@pytest.mark.parametrize("case", CASES[1:8], ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_gradients_are_the_turn_back(case, dtype):
    import flash_attn2_b200 as fa2

    b, s, h, hk, d, sections, ia, ip = case
    q, k, positions, inv_freq = _inputs(4, b, s, h, hk, d, sections, dtype)
    dq, dk, _, _ = _inputs(5, b, s, h, hk, d, sections, dtype)
    qc, kc = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    out = fa2.rotary_axes_func(qc, kc, positions.cuda(), inv_freq.cuda(), sections, ia, ip)
    for g, x in zip(torch.autograd.grad(out, (qc, kc), (dq.cuda(), dk.cuda())), (dq, dk)):
        torch.testing.assert_close(g.cpu().double(), turn(x, positions, inv_freq, sections, ia, ip, inverse=True), **turn_tolerance(x, dtype))


def test_gradients_against_differences():
    """The turn is linear: <g, turn(x + h e) - turn(x)> / h = <grad, e> for any h, up to the outputs' roundings."""
    import flash_attn2_b200 as fa2

    b, s, h, hk, d, sections = 1, 9, 2, 1, 32, (6, 5, 5)
    q, k, positions, inv_freq = (t.cuda() for t in _inputs(6, b, s, h, hk, d, sections, torch.float16))
    g = torch.randn_like(q)
    x = q.clone().requires_grad_()
    grad, = torch.autograd.grad(fa2.rotary_axes_func(x, k, positions, inv_freq, sections)[0], x, g)
    gen = torch.Generator().manual_seed(1)
    for _ in range(10):
        e = torch.zeros_like(q)
        i = int(torch.randint(0, q.numel(), (1,), generator=gen))
        e.view(-1)[i] = 8.0
        hi, lo = (fa2.rotary_axes_func(q + sign * e, None, positions, inv_freq, sections)[0].double() for sign in (1, -1))
        want = ((hi - lo) * g.double()).sum() / 16
        # outputs of magnitude 12, two of them, off by 2^-11 of it each, on both sides, and x + e by as much; over a step of 16
        assert abs(grad.view(-1)[i].double() - want) <= 8 * 12 * 2.0 ** -11 * float(g.abs().max()) / 16 + 2.0 ** -11 * float(grad.abs().max())


def test_gradients_of_shared_heads_sums_and_unused_outputs():
    import flash_attn2_b200 as fa2

    b, s, h, hk, d, sections = 2, 21, 6, 6, 64, (12, 10, 10)
    q, k, positions, inv_freq = (t.cuda() for t in _inputs(7, b, s, h, hk, d, sections, torch.bfloat16))
    shared = k[:, :, :1].clone().requires_grad_()          # one key head for all: its gradient is their sum
    out = fa2.rotary_axes_func(q, shared.expand(b, s, hk, d), positions, inv_freq, sections)
    grad, = torch.autograd.grad(out[1], shared, torch.ones_like(out[1]))
    want = turn(torch.ones(b, s, 1, d), positions.cpu(), inv_freq.cpu(), sections, inverse=True) * hk
    torch.testing.assert_close(grad.cpu().double(), want, rtol=2 ** -7, atol=hk * 2 ** -7)
    x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
    a, c = fa2.rotary_axes_func(x, y, positions, inv_freq, sections)
    a.sum().backward()                                      # an expanded gradient, and none for the keys
    assert y.grad is None or not y.grad.any()
    torch.testing.assert_close(x.grad.cpu().double(), turn(torch.ones(b, s, h, d), positions.cpu(), inv_freq.cpu(), sections, inverse=True),
                               rtol=2 ** -8 * 1.001, atol=1e-5)
    a, c = fa2.rotary_axes_func(q, y, positions, inv_freq, sections)
    assert c.requires_grad
    y.grad = None
    c.backward(torch.ones_like(c))
    assert y.grad is not None


def test_second_order():
    """The gradient is a turn, and has gradients itself."""
    import flash_attn2_b200 as fa2

    q, k, positions, inv_freq = (t.cuda() for t in _inputs(8, 1, 12, 2, 2, 64, (32,), torch.float16))
    x, g = q.clone().requires_grad_(), torch.randn_like(q).requires_grad_()
    out = fa2.rotary_axes_func(x, None, positions, inv_freq, (32,))[0]
    grad, = torch.autograd.grad(out, x, g, create_graph=True)
    second, = torch.autograd.grad(grad, g, k)
    torch.testing.assert_close(second.cpu().double(), turn(k.cpu(), positions.cpu(), inv_freq.cpu(), (32,)), **turn_tolerance(k, torch.float16))


def test_positions_that_change_before_the_backward_are_noticed():
    import flash_attn2_b200 as fa2

    q, k, positions, inv_freq = (t.cuda() for t in _inputs(9, 1, 12, 2, 2, 64, (32,), torch.float16))
    out = fa2.rotary_axes_func(q.requires_grad_(), k, positions, inv_freq, (32,))[0]
    positions += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_refusals():
    import torch.autograd.forward_ad as fwd_ad

    import flash_attn2_b200 as fa2

    q, k, positions, inv_freq = (t.cuda() for t in _inputs(10, 2, 12, 4, 2, 64, (12, 10, 10), torch.bfloat16))
    sections = (12, 10, 10)

    def refused(kind, **kw):
        args = dict(q=q, k=k, positions=positions, inv_freq=inv_freq, sections=sections)
        args.update(kw)
        with pytest.raises(kind):
            fa2.rotary_axes_func(**args)

    refused(TypeError, k=k.half())
    refused(TypeError, q=q.float(), k=k.float())
    refused(TypeError, positions=positions.float())
    refused(TypeError, inv_freq=inv_freq.double())
    refused(TypeError, interleaved_axes=1)
    refused(ValueError, k=k[:, :5])
    refused(ValueError, k=k[..., :32])
    refused(ValueError, q=q[0, 0], k=None)
    refused(ValueError, positions=positions[:2])
    refused(ValueError, positions=positions[:, :1])
    refused(ValueError, positions=positions[:, :, :5])
    refused(ValueError, inv_freq=inv_freq[:31])
    refused(ValueError, sections=(12, 10))
    refused(ValueError, sections=(2, 10, 20), interleaved_axes=True)
    refused(ValueError, q=q[..., :60], k=k[..., :60], sections=(30,), positions=positions[:1], inv_freq=inv_freq[:30])
    refused(NotImplementedError, positions=positions.cpu())
    refused(RuntimeError, inv_freq=inv_freq.clone().requires_grad_())
    with fwd_ad.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
        fa2.rotary_axes_func(fwd_ad.make_dual(q, q), k, positions, inv_freq, sections)
    with pytest.raises(RuntimeError, match="transform"):
        torch.func.vmap(lambda x: fa2.rotary_axes_func(x, k, positions, inv_freq, sections)[0])(torch.stack([q, q]))
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: fa2.rotary_axes_func(x, k, positions, inv_freq, sections)[0], q)


def test_before_the_packed_and_dense_attention():
    """Turned queries and keys go into the attention, and the gradients come back through both."""
    import flash_attn2_b200 as fa2
    from oracle.attention_oracle import attention_forward

    b, s, h, hk, d, sections = 2, 150, 4, 2, 64, (12, 10, 10)
    q, k, positions, inv_freq = _inputs(11, b, s, h, hk, d, sections, torch.bfloat16)
    v = torch.randn(b, s, hk, d, generator=torch.Generator().manual_seed(1)).bfloat16()
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    tq, tk = fa2.rotary_axes_func(leaves[0], leaves[1], positions.cuda(), inv_freq.cuda(), sections)
    out = fa2.flash_attn_func(tq, tk, leaves[2], causal=True)
    want, _ = attention_forward(tq.detach().cpu(), tk.detach().cpu(), v, causal=True)
    torch.testing.assert_close(out.float().cpu(), want, atol=1e-2, rtol=5e-2)
    seen = torch.autograd.grad(fa2.flash_attn_func(*(t.detach().requires_grad_() for t in (tq, tk)), leaves[2], causal=True).sum(), leaves[2])
    grads = torch.autograd.grad(out.sum(), leaves)
    assert torch.equal(grads[2], seen[0]) and all(g.isfinite().all() and g.any() for g in grads)


GRAPHS = r"""
import sys
sys.path[:0] = ["kernels-community-rs_b200"]
import torch
import flash_attn2_b200 as fa2
q = torch.randn(1, 64, 4, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
pos = torch.arange(64, device="cuda").view(1, 1, 64)
freq = torch.rand(32, device="cuda")
g = torch.randn_like(q)
rotary = lambda: fa2.rotary_axes_func(q, None, pos, freq, (32,))[0]
f = rotary if sys.argv[1] == "rotary" else lambda: torch.sin(q)
want, = torch.autograd.grad(f(), q, g)
if sys.argv[2] == "beside":
    eager = f()                  # lives while a pass over the same leaf is captured
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
try:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got, = torch.autograd.grad(f(), q, g)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    print("captured")
except RuntimeError as e:
    print("refused")
torch.cuda.synchronize()
f().backward(g)
torch.cuda.synchronize()
assert torch.equal(q.grad, want)
print("done")
"""


def _captured(*args):
    run = subprocess.run([sys.executable, "-c", GRAPHS, *args], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr[-2000:]
    return run.stdout.split()


def test_a_captured_backward():
    assert _captured("rotary", "alone") == ["captured", "done"]


def test_a_captured_backward_beside_an_eager_graph_of_the_same_leaf():
    """torch's engine refuses that for any operation (the leaf's node belongs to the eager stream). An error, and nothing worse: the
    process goes on."""
    got = _captured("rotary", "beside")
    assert got == _captured("sin", "beside") and got[-1] == "done"


@pytest.mark.parametrize("d,sections,pad", [(128, (16, 24, 24), 0), (128, (16, 24, 24), 3), (96, (8, 12, 12), 0), (72, (3, 4, 5, 8), 0), (248, (44, 41, 39), 0)])
@pytest.mark.parametrize("interleaved_pairs", [False, True])
def test_in_place(d, sections, pad, interleaved_pairs):
    """The C entry point with q_out = q and k_out = k, on tensors that 16-byte loads can take and on others (rows at odd strides, pairs that
    are no multiple of 8): the bits of a call with other outputs, also where a call is long enough for many warps of a token."""
    import ctypes as C

    import flash_attn2_b200 as fa2
    from flash_attn2_b200 import _cabi

    b, s, h, hk = 2, 333, 24, 3
    q, k, positions, inv_freq = (t.cuda() for t in _inputs(8, b, s, h, hk, d, sections, torch.bfloat16))
    q, k = (torch.nn.functional.pad(t, (0, pad))[..., :d] for t in (q, k))
    want = fa2.rotary_axes_func(q, k, positions, inv_freq, sections, interleaved_pairs=interleaved_pairs)
    a = _cabi.RotaryArgs(size=C.sizeof(_cabi.RotaryArgs), q=q.data_ptr(), q_out=q.data_ptr(), k=k.data_ptr(), k_out=k.data_ptr(), q_stride=q.stride()[:3],
                         q_out_stride=q.stride()[:3], k_stride=k.stride()[:3], k_out_stride=k.stride()[:3], positions=positions.data_ptr(),
                         position_stride=positions.stride(), inv_freq=inv_freq.data_ptr(), position_bits=64, dtype=_cabi.FA2_BF16, batch=b, seqlen=s,
                         heads=h, heads_k=hk, head_dim=d, axes=len(sections), sections=tuple(sections) + (0,) * (4 - len(sections)),
                         interleaved_pairs=interleaved_pairs)
    assert positions.dtype == torch.int64
    _cabi.check(_cabi.load().fa2_rotary(C.byref(a), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
