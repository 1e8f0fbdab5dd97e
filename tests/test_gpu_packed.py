"""flash_attention_packed on the GPU, forward and gradients, against the formulas in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from flash_attention_triton_b200 import _lib, flash_attention_packed, flash_attention_v2
from packed_helpers import exact_packed

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
RAGGED = [1, 0, 127, 128, 129, 300, 2, 0, 64]


@pytest.fixture(autouse=True)
def _no_status():
    yield
    assert _lib.device_status() == 0


def cu_of(lengths, first=0):
    return torch.tensor([first, *(first + torch.tensor(lengths).cumsum(0)).tolist()], dtype=torch.int32, device="cuda")


def inputs(lengths, heads, kv_heads, d, dtype, seed=0, behind=0, peak=1.0, junk=math.nan):
    """q, k, v, dO with `junk` in the rows behind the last sequence."""
    g = torch.Generator().manual_seed(seed)
    rows = sum(lengths)
    out = []
    for h, mul in ((heads, peak), (kv_heads, peak), (kv_heads, 1.0), (heads, 1.0)):
        t = torch.full((rows + behind, h, d), junk)
        t[:rows] = torch.randn(rows, h, d, generator=g) * mul
        out.append(t.to(dtype).cuda())
    return out


def run(q, k, v, cu, do=None, scale=None):
    if do is None:
        with torch.no_grad():
            return {"o": flash_attention_packed(q, k, v, cu, scale)}
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = flash_attention_packed(*leaves, cu, scale)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))


def check(lengths, heads, kv_heads, d, dtype, behind=0, peak=1.0, scale=None, seed=0):
    q, k, v, do = inputs(lengths, heads, kv_heads, d, dtype, seed, behind, peak)
    got = run(q, k, v, cu_of(lengths), do, scale)
    rows = sum(lengths)
    want = exact_packed(*(t[:rows] for t in (q, k, v)), lengths, do[:rows], scale)
    for name, (value, tolerance) in want.items():
        off = (got[name][:rows].double() - value).abs()
        assert (off <= tolerance).all(), f"{name}: {(off / tolerance).max().item():.3g} times the bound, {off.max().item():.3g}"
        assert (got[name][rows:] == 0).all(), name
        assert got[name].is_contiguous() and got[name].dtype == dtype
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 96, 104, 128])
def test_head_dims(dtype, d):
    check(RAGGED, 4, 2, d, dtype, behind=50)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (2, 1), (3, 1), (6, 2), (10, 2), (8, 1), (16, 8), (32, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_head_layouts(heads, kv_heads, d):
    check([200, 1, 129], heads, kv_heads, d, BF16)


@pytest.mark.parametrize("lengths", [[1], [1] * 300, [128] * 9, [129] * 9, [64] * 40, [0, 0, 5], [0], [1000, 1, 1], [700], [2048, 130, 1500],
                                     list(range(60)), [384, 385, 511, 513]])
@pytest.mark.parametrize("heads,kv_heads,d,dtype", [(4, 2, 64, FP16), (3, 1, 128, BF16)])
def test_lengths(lengths, heads, kv_heads, d, dtype):
    check(lengths, heads, kv_heads, d, dtype, behind=3)


@pytest.mark.parametrize("lengths,heads,kv_heads", [([900, 40, 1300, 333], 32, 16), ([5000, 300], 8, 4)])
@pytest.mark.parametrize("d", [32, 64])
def test_steps_of_64_rows(lengths, heads, kv_heads, d):
    """Enough tiles that the backward takes the form with two CTAs on an SM."""
    check(lengths, heads, kv_heads, d, FP16)
    check(lengths, heads, kv_heads, d, BF16)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_peaked(dtype):
    check([300, 77, 513], 4, 2, 64, dtype, peak=3.0, scale=0.5)


@pytest.mark.parametrize("size", [1e-4, 1e3])
def test_gradients_of_any_size_at_fp16(size):
    lengths = [300, 77]
    q, k, v, do = inputs(lengths, 4, 2, 64, FP16)
    power = 2 ** round(math.log2(size))
    one = run(q, k, v, cu_of(lengths), do.double().mul(2.0**-4).to(FP16))
    many = run(q, k, v, cu_of(lengths), do.double().mul(2.0**-4 * power).to(FP16))
    # Powers of two of dO leave every rounding where it was, but for numbers below fp16's normal ones, in dO and in the
    # results, which are off by 2^-25 at most where dO is the smaller one.  From dO that reaches dV through a column of weights
    # (their sum is dV of dO = 1), and dQ and dK through dP and delta: scale P (sum |v| + sum |o|) |k|, summed over a row of
    # weights (1), or |q| over a column of them.  Where such a difference moves a result across the middle of two numbers, the
    # two roundings are half a step apart each, 2^-11 twice.
    off = 2.0**-25 * max(1.0, power)
    column = run(q, k, v, cu_of(lengths), torch.ones_like(do))["dv"].max().item() * (1 + 2.0**-8)
    through = 64**-0.5 * 2 * 64 * v.double().abs().max().item()
    reach = {"dv": column, "dq": through * k.double().abs().max().item(), "dk": through * q.double().abs().max().item() * column}
    for n in ("dq", "dk", "dv"):
        a, b = one[n].double() * power, many[n].double()
        assert ((a - b).abs() <= 2 * 2.0**-11 * a.abs() + off * (reach[n] + 1)).all(), n


def test_one_sequence_has_the_bits_of_the_dense_operator():
    """The same arithmetic in the same order, at a head dim and length whose dense forward takes 128-row KV tiles."""
    q, k, v, _ = inputs([1500], 4, 4, 128, BF16)
    dense = flash_attention_v2(*(t.transpose(0, 1)[None] for t in (q, k, v)))
    assert torch.equal(run(q, k, v, cu_of([1500]))["o"], dense[0].transpose(0, 1))


def test_a_sequence_does_not_depend_on_its_neighbours():
    """NaN and infinities in the other sequences, and another place among them, change no bit."""
    lengths = [130, 200, 70, 257]
    for heads, kv_heads, d, dtype in ((4, 2, 64, BF16), (3, 1, 128, FP16)):
        q, k, v, do = inputs(lengths, heads, kv_heads, d, dtype)
        clean = run(q, k, v, cu_of(lengths), do)
        for other, junk in ((0, math.nan), (2, math.inf), (3, -math.inf), (1, math.nan)):
            first = sum(lengths[:other])
            rows = slice(first, first + lengths[other])
            spoilt = [t.clone() for t in (q, k, v, do)]
            for t in spoilt:
                t[rows] = junk
            got = run(*spoilt[:3], cu_of(lengths), spoilt[3])
            for n in got:
                keep = torch.ones(sum(lengths), dtype=torch.bool)
                keep[rows] = False
                assert torch.equal(got[n][keep], clean[n][keep]), (n, other)
        for s in range(4):  # alone
            first = sum(lengths[:s])
            rows = slice(first, first + lengths[s])
            alone = run(*(t[rows].clone() for t in (q, k, v)), cu_of([lengths[s]]), do[rows].clone())
            for n in alone:
                assert torch.equal(alone[n], clean[n][rows]), (n, s)


def test_later_rows_do_not_change_earlier_ones():
    """Bit by bit outside the 32 rows that decide together when to rescale; those keep their value within its bound."""
    q, k, v, _ = inputs([400], 4, 2, 64, BF16)
    a = run(q, k, v, cu_of([400]))["o"]
    want, tolerance = exact_packed(q, k, v, [400])["o"]
    k[300:], v[300:] = 7.0, -3.0
    b = run(q, k, v, cu_of([400]))["o"]
    assert torch.equal(a[:288], b[:288]) and not torch.equal(a[300:], b[300:])
    assert ((b[:300].double() - want[:300]).abs() <= tolerance[:300]).all()


def test_row_without_a_finite_score_has_no_softmax():
    q, k, v, _ = inputs([200, 150], 2, 1, 64, BF16)
    q, k = q.abs(), k.abs()
    k[0] = -math.inf
    o = run(q, k, v, cu_of([200, 150]))["o"]
    assert o[0].isnan().all() and o[1:].isfinite().all()


def test_rows_in_front_and_behind():
    lengths = [40, 100]
    q, k, v, do = inputs(lengths, 4, 2, 64, BF16)
    want = run(q, k, v, cu_of(lengths), do)
    pad = [torch.cat([torch.full_like(t[:30], math.nan), t, torch.full_like(t[:90], math.nan)]) for t in (q, k, v, do)]
    got = run(*pad[:3], cu_of(lengths, 30), pad[3])
    for n in got:
        assert torch.equal(got[n][30:170], want[n]) and (got[n][:30] == 0).all() and (got[n][170:] == 0).all(), n


def test_no_rows():
    t = torch.zeros(0, 2, 64, dtype=BF16, device="cuda", requires_grad=True)
    o = flash_attention_packed(t, t, t, cu_of([0, 0]))
    (g,) = torch.autograd.grad(o, [t], o.detach())
    assert o.shape == g.shape == (0, 2, 64)


@pytest.mark.parametrize("cu", [[0, 50, 40, 100], [0, 50, 101], [-1, 50, 100], [5, 3], [2**31 - 1, 2**31 - 1]])
def test_sequences_that_fall_or_leave_the_rows(cu):
    q, k, v, do = inputs([100], 4, 2, 64, BF16)
    got = run(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), do)
    assert _lib.device_status() == 0x80000
    for n in got:
        assert (got[n] == 0).all(), n


def test_strided_inputs():
    lengths = [150, 90]
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(240, 4 + 2 + 2, 64, generator=g).to(BF16).cuda()
    do = torch.randn(4, 240, 64, generator=g).to(BF16).cuda().transpose(0, 1)  # heads first
    views = fused.split([4, 2, 2], 1)
    want = run(*(t.contiguous() for t in views), cu_of(lengths), do.contiguous())
    got = run(*views, cu_of(lengths), do)
    leaf = fused.clone().requires_grad_(True)
    o = flash_attention_packed(*leaf.split([4, 2, 2], 1), cu_of(lengths))
    (grad,) = torch.autograd.grad(o, [leaf], do)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    assert torch.equal(grad, torch.cat([want["dq"], want["dk"], want["dv"]], 1))
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in views]
    odd = [torch.nn.functional.pad(t, (0, 4))[..., :64] for t in views]  # rows 8 bytes apart from 16-byte boundaries
    assert torch.equal(run(*heads_first, cu_of(lengths))["o"], want["o"]) and torch.equal(run(*odd, cu_of(lengths))["o"], want["o"])
    flat = torch.cat([fused.new_zeros(1), fused.flatten()])[1:]  # dense, 2 bytes behind a 16-byte boundary
    odd = [flat.view(240, 8, 64)[:, a:b] for a, b in ((0, 4), (4, 6), (6, 8))]
    assert torch.equal(run(*odd, cu_of(lengths))["o"], want["o"])
    assert torch.equal(run(*odd, cu_of(lengths), torch.cat([do.new_zeros(1), do.contiguous().flatten()])[1:].view(240, 4, 64))["dk"], want["dk"])
    one = do[:, :1].expand(-1, 4, -1)  # a broadcast gradient
    a, b = run(*views, cu_of(lengths), one), run(*views, cu_of(lengths), one.contiguous())
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_heads_that_share_a_leaf_and_unused_gradients():
    lengths = [100, 30]
    q, k, v, do = inputs(lengths, 4, 2, 64, BF16)
    want = run(q, k, v, cu_of(lengths), do)
    k.requires_grad_(True)
    o = flash_attention_packed(q, k, v, cu_of(lengths))
    (dk,) = torch.autograd.grad(o, [k], do)
    assert torch.equal(dk, want["dk"])
    shared = v.clone().requires_grad_(True)  # keys and values are one tensor
    a = flash_attention_packed(q, shared, shared, cu_of(lengths))
    (both,) = torch.autograd.grad(a, [shared], do)
    apart = run(q, v, v, cu_of(lengths), do)
    assert torch.equal(both, apart["dk"] + apart["dv"])


def test_no_second_derivative():
    q, k, v, do = inputs([50], 2, 1, 64, BF16)
    q.requires_grad_(True)
    o = flash_attention_packed(q, k, v, cu_of([50]))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(o, [q], do, create_graph=True)


def test_gradient_against_differences():
    """Along the gradient itself, with the kernel's own forward: the difference of sum(o dO) over a step that moves it well
    above the roundings of o."""
    lengths = [300, 77, 130]
    q, k, v, do = inputs(lengths, 4, 2, 64, FP16, seed=4)
    grads = run(q, k, v, cu_of(lengths), do)
    for i, name in enumerate(("dq", "dk", "dv")):
        x, g = (q, k, v)[i], grads[name].double()
        step = 0.05 / g.abs().max()
        ends, at = [], []
        for sign in (1, -1):
            moved = [q, k, v]
            moved[i] = (x.double() + sign * step * g).to(FP16)
            at.append(moved[i].double())
            ends.append((run(*moved, cu_of(lengths))["o"].double() * do.double()).sum().item())
        predicted = (g * (at[0] - at[1])).sum().item()  # the step as it was rounded
        assert abs((ends[0] - ends[1]) / predicted - 1) < 0.05, name


def test_repeats_have_the_same_bits():
    lengths = [700, 3, 1200, 90]
    q, k, v, do = inputs(lengths, 8, 2, 128, BF16)
    first = run(q, k, v, cu_of(lengths), do)
    for _ in range(5):
        again = run(q, k, v, cu_of(lengths), do)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_many_rows_and_sequences():
    """More tiles than the plan has bins for one sequence's, and more sequences than one round of its threads."""
    g = torch.Generator().manual_seed(3)
    lengths = [140000, *torch.randint(0, 40, (1500,), generator=g).tolist()]
    q, k, v, _ = inputs(lengths, 1, 1, 32, FP16)
    o = run(q, k, v, cu_of(lengths))["o"]
    first = 140000
    want = exact_packed(q[first:], k[first:], v[first:], lengths[1:])["o"]
    assert ((o[first:].double() - want[0]).abs() <= want[1]).all()
    dense = flash_attention_v2(*(t[:first].transpose(0, 1)[None] for t in (q, k, v)))
    assert torch.equal(o[:first], dense[0].transpose(0, 1))


def test_on_another_stream_and_captured():
    lengths = [200, 90]
    q, k, v, do = inputs(lengths, 4, 2, 64, BF16, behind=100, junk=0.5)
    cu = cu_of(lengths)
    want = run(q, k, v, cu, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, cu, do)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(q, k, v, cu, do)
    for lengths in ([200, 90], [10, 0], [1, 389], [0, 0], [200, 90]):  # the graph follows cu_seqlens
        cu.copy_(cu_of(lengths))
        graph.replay()
        want = run(q, k, v, cu_of(lengths), do)
        assert all(torch.equal(got[n], want[n]) for n in want), lengths


def test_two_streams_at_once():
    sets = [inputs([500, 20, 300], 8, 2, 64, BF16, seed=s) for s in (1, 2)]
    cu = cu_of([500, 20, 300])
    want = [run(*t[:3], cu, t[3]) for t in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for t, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append(run(*t[:3], cu, t[3]))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(a[n], b[n]) for n in b)


def test_status_check_raises(monkeypatch):
    q, k, v, _ = inputs([20], 2, 1, 64, BF16)
    monkeypatch.setenv("FA2_B200_CHECK_STATUS", "1")
    flash_attention_packed(q, k, v, cu_of([20]))
    with pytest.raises(_lib.Fa2Error, match="status 0x80000"):
        flash_attention_packed(q, k, v, cu_of([21]))


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_on_the_other_device():
    q, k, v, do = inputs([100, 30], 4, 2, 64, BF16)
    want = run(q, k, v, cu_of([100, 30]), do)
    got = run(*(t.to("cuda:1") for t in (q, k, v)), cu_of([100, 30]).to("cuda:1"), do.to("cuda:1"))
    assert all(torch.equal(got[n].cpu(), want[n].cpu()) for n in want)


def test_saved_tensor_hooks():
    """Saved tensors may leave the GPU and come back; one that comes back changed is refused."""
    lengths = [90, 40]
    q, k, v, do = inputs(lengths, 4, 2, 64, BF16)
    want = run(q, k, v, cu_of(lengths), do)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    with torch.autograd.graph.save_on_cpu():
        o = flash_attention_packed(*leaves, cu_of(lengths))
    assert all(torch.equal(a, want[n]) for n, a in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:-1]):
        o = flash_attention_packed(*leaves, cu_of(lengths))
    with pytest.raises(RuntimeError, match="have changed"):
        torch.autograd.grad(o, leaves, do)
    o = flash_attention_packed(*leaves, cu_of(lengths))
    with torch.no_grad():
        k.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o, leaves, do)


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 4, 64), (9, 3, 40), (5, 5, 128), (2, 1, 32)])
@pytest.mark.parametrize("lengths", [[700, 1, 300, 129, 640, 0, 128, 90, 1500, 2], [257] * 32, [2900, 64], [1] * 31 + [2500]])
def test_items_found_with_and_without_a_plan(heads, kv_heads, d, lengths):
    """With up to 32 sequences and few items the CTAs find these themselves, one or several each; with 40 a plan has them: the same bits."""
    check(lengths, heads, kv_heads, d, BF16)
    q, k, v, do = inputs(lengths, heads, kv_heads, d, BF16, behind=7)
    o = run(q, k, v, cu_of(lengths))["o"]
    assert torch.equal(o, run(q, k, v, cu_of(lengths + [0] * (40 - len(lengths))))["o"])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (6, 2), (8, 2), (12, 2), (16, 1)])
def test_query_heads_shared_by_a_cluster(dtype, d, heads, kv_heads):
    """Four, two or one CTA to a key head's tile, by the query heads that there are."""
    check([300, 1, 129, 0, 128, 450], heads, kv_heads, d, dtype, behind=3)


def test_calls_one_behind_the_other():
    """Kernels of one call start under those of the call before it, in memory that calls before that one have given back."""
    sets = [([500 + 40 * i, 3, 129], *shape) for i, shape in enumerate([(8, 2, 64), (8, 4, 128), (3, 3, 32), (16, 1, 64), (4, 2, 128)])]
    data = [(*inputs(lengths, h, hk, d, BF16, seed=i), cu_of(lengths)) for i, (lengths, h, hk, d) in enumerate(sets)]
    want = []
    for q, k, v, do, cu in data:
        want.append(run(q, k, v, cu, do))
        torch.cuda.synchronize()
    for _ in range(6):
        got = [run(q, k, v, cu, do) for q, k, v, do, cu in data * 3]
        for i, g in enumerate(got):
            assert all(torch.equal(g[n], want[i % len(data)][n]) for n in g), i
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [run(q, k, v, cu, do) for q, k, v, do, cu in data * 2]
    for _ in range(5):
        for g in got:
            for t in g.values():
                t.zero_()
        graph.replay()
        for i, g in enumerate(got):
            assert all(torch.equal(g[n], want[i % len(data)][n]) for n in g), i


def test_offsets_beyond_32_bits():
    """2.3e9 elements in q and its gradient."""
    lengths, heads, d = [128] * 4400 + [77], 32, 128
    rows = sum(lengths)
    q, do = (torch.randn(rows, heads, d, device="cuda", dtype=BF16) for _ in range(2))
    k, v = (torch.randn(rows, 1, d, device="cuda", dtype=BF16) for _ in range(2))
    got = run(q, k, v, cu_of(lengths), do)
    for first, of in ((0, lengths[:2]), (rows - 205, lengths[-2:])):
        part = slice(first, first + sum(of))
        for name, (value, tolerance) in exact_packed(*(t[part] for t in (q, k, v)), of, do[part], None).items():
            assert ((got[name][part].double() - value).abs() <= tolerance).all(), (name, first)
