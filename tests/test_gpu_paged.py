"""append_kv_cache and flash_attention_decode on the GPU, against their formulas in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from flash_attention_triton_b200 import _lib
from paged_helpers import Cache, cu_seqlens_of, decode_tolerance, exact_decode, fa, rotated, rotation_tolerance

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _no_status():
    yield
    assert _lib.device_status() == 0


def normal(*shape, dtype, seed=1):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# ------------------------------------------------------------------------------------------------ append
def check_append(held, new, page, heads, kv_heads, d, dtype, rotary, interleaved=False, layout="slots", tokens_only=False,
                 behind=0, seed=3):
    """Appends to sequences that hold `held` positions, and looks at every slot of the cache."""
    total = [a + b for a, b in zip(held, new)]
    cache = Cache(held, total, page, kv_heads, d, dtype, seed, layout)
    rows = sum(new) + behind
    q, k, v = normal(rows, heads, d, dtype=dtype, seed=1), normal(rows, kv_heads, d, dtype=dtype, seed=2), normal(rows, kv_heads, d, dtype=dtype, seed=3)
    cos, sin = fa.rotary_tables(max(total) + 1, rotary, device="cuda") if rotary else (None, None)
    before = cache.k.clone(), cache.v.clone()
    cu = None if tokens_only else cu_seqlens_of(new)
    q_out, k_out = fa.append_kv_cache(k, v, cache.k, cache.v, cache.table, cache.lengths(total), cu_seqlens=cu, q=q, cos=cos, sin=sin,
                                      interleaved=interleaved, return_k=True)
    row = 0
    for s, n in enumerate(new):
        if n == 0:
            continue
        positions = torch.arange(held[s], total[s], device="cuda")
        at = cache.places(s, range(held[s], total[s]))
        for x, out in ((q, q_out), (k, k_out)):
            x, got = x[row : row + n], out[row : row + n].double()
            want = rotated(x, cos, sin, positions, interleaved)
            assert ((got - want).abs() <= rotation_tolerance(dtype, want, x)).all()
            if rotary < d:
                assert torch.equal(out[row : row + n, :, rotary:], x[:, :, rotary:])
        assert torch.equal(cache.k[at], k_out[row : row + n])
        assert torch.equal(cache.v[at], v[row : row + n])
        before[0][at], before[1][at] = cache.k[at], cache.v[at]
        row += n
    for now, was in zip((cache.k, cache.v), before):  # every other slot has the bits it had
        assert torch.equal(now.contiguous().view(torch.int16), was.contiguous().view(torch.int16))
    assert (q_out[row:] == 0).all() and (k_out[row:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d,rotary,interleaved", [(64, 64, False), (128, 128, False), (128, 64, False), (80, 80, True),
                                                  (80, 48, False), (72, 16, True), (8, 0, False), (256, 256, False), (40, 32, False)])
def test_append_prompts(dtype, d, rotary, interleaved):
    check_append([0, 5, 0, 130], [37, 1, 0, 70], 16, 6, 2, d, dtype, rotary, interleaved, behind=9)


@pytest.mark.parametrize("page", [1, 7, 16, 64, 200])
@pytest.mark.parametrize("layout", ["slots", "heads"])
def test_append_single_tokens(page, layout):
    held = [0, 1, 15, 16, 17, 100, 199, 200]
    check_append(held, [1] * 8, page, 4, 4, 64, BF16, 64, layout=layout, tokens_only=True)


@pytest.mark.parametrize("batch,heads,kv_heads,d", [(1, 1, 1, 8), (300, 32, 8, 128), (700, 2, 1, 64), (5, 160, 8, 128)])
def test_append_many(batch, heads, kv_heads, d):
    g = torch.Generator().manual_seed(batch)
    held = torch.randint(0, 40, (batch,), generator=g).tolist()
    check_append(held, [1] * batch, 16, heads, kv_heads, d, FP16, d // 16 * 16, tokens_only=True)


@pytest.mark.parametrize("batch", [1, 2, 31, 32, 33, 150])
def test_append_finds_the_sequences(batch):
    """Sequences without tokens before, between and behind those that have some; up to 32 are looked up at once."""
    g = torch.Generator().manual_seed(batch)
    new = [n * (torch.rand(1, generator=g).item() < 0.6) for n in torch.randint(1, 50, (batch,), generator=g).tolist()]
    new[batch // 2] = 61
    check_append(torch.randint(0, 40, (batch,), generator=g).tolist(), new, 16, 4, 2, 64, BF16, 64, behind=5)


def test_append_long_prompt_and_far_positions():
    check_append([100000, 0], [300, 1500], 64, 2, 1, 64, BF16, 64)


def test_append_leaves_out_what_has_no_place():
    """Empty places of a batch, prompts longer than their sequence, page numbers and positions outside."""
    cache = Cache([4, 4, 4, 4], [16, 16, 16, 16], 4, 2, 64, BF16)
    k, v = normal(4, 2, 64, dtype=BF16), normal(4, 2, 64, dtype=BF16, seed=2)
    before = cache.k.clone()
    _, k_out = fa.append_kv_cache(k, v, cache.k, cache.v, cache.table, cache.lengths([0, 5, -3, 0]), return_k=True)
    assert _lib.device_status() == 0
    assert (k_out[[0, 2, 3]] == 0).all() and torch.equal(k_out[1], k[1])
    at = cache.places(1, [4])
    assert torch.equal(cache.k[at][0], k[1])
    before[at] = cache.k[at]
    assert torch.equal(cache.k.view(torch.int16), before.view(torch.int16))
    # five rows of a sequence of three positions: the first two rows have no place
    cu = torch.tensor([0, 4, 4, 4, 4], dtype=torch.int32, device="cuda")
    _, k_out = fa.append_kv_cache(k, v, cache.k, cache.v, cache.table, cache.lengths([2, 4, 4, 4]), cu_seqlens=cu, return_k=True)
    assert (k_out[:2] == 0).all() and torch.equal(k_out[2:], k[2:]) and torch.equal(cache.k[cache.places(0, [0, 1])], k[2:])
    before = cache.k.clone()
    table = cache.table.clone()
    table[0, 1], table[1, 1] = -1, cache.k.shape[0]
    cos, sin = fa.rotary_tables(6, 64, device="cuda")
    for lengths in ([5, 0, 0, 0], [0, 6, 0, 0], [0, 0, 17, 0], [0, 0, 0, 7], [0, 0, 2**31 - 1, 0]):
        _, k_out = fa.append_kv_cache(k, v, cache.k, cache.v, table, cache.lengths(lengths), cos=cos, sin=sin, return_k=True)
        assert _lib.device_status() == 0x40001
        assert (k_out == 0).all() and torch.equal(cache.k.view(torch.int16), before.view(torch.int16))


def test_append_strided_inputs():
    fused = normal(50, 4 + 2 + 2, 64, dtype=BF16)
    q, k, v = fused.split([4, 2, 2], 1)
    cache, plain = (Cache([0, 0], [30, 20], 16, 2, 64, BF16) for _ in range(2))
    cos, sin = fa.rotary_tables(40, 64, device="cuda")
    a = fa.append_kv_cache(k, v, cache.k, cache.v, cache.table, cache.lengths([30, 20]), cu_seqlens=cu_seqlens_of([30, 20]), q=q, cos=cos, sin=sin)
    b = fa.append_kv_cache(k.contiguous(), v.contiguous(), plain.k, plain.v, plain.table, plain.lengths([30, 20]),
                           cu_seqlens=cu_seqlens_of([30, 20]), q=q.contiguous(), cos=cos, sin=sin)
    assert torch.equal(a[0], b[0]) and a[1] is None and b[1] is None
    for x, y in ((cache.k, plain.k), (cache.v, plain.v)):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    # rows that no kernel can read in place: a stride of 8 bytes more, columns apart
    odd = normal(50, 2, 68, dtype=BF16)[..., :64]
    wide = normal(50, 2, 128, dtype=BF16)[..., ::2]
    odd = torch.cat([odd.new_zeros(1), odd.contiguous().flatten()])[1:].view(50, 2, 64)  # dense, 2 bytes behind a boundary
    fa.append_kv_cache(odd, wide, cache.k, cache.v, cache.table, cache.lengths([30, 20]), cu_seqlens=cu_seqlens_of([30, 20]))
    assert torch.equal(cache.k[cache.places(0, range(30))], odd[:30]) and torch.equal(cache.v[cache.places(1, range(20))], wide[30:])


def test_append_nothing():
    cache = Cache([3], [8], 4, 2, 64, BF16)
    empty = torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    q, k = fa.append_kv_cache(empty, empty, cache.k, cache.v, cache.table, cache.lengths(), cu_seqlens=cu_seqlens_of([0]), q=empty, return_k=True)
    assert q.shape == k.shape == (0, 2, 64)


def test_append_marks_the_cache_as_written():
    cache = Cache([0], [8], 4, 2, 64, BF16)
    was = cache.k._version
    k = normal(1, 2, 64, dtype=BF16)
    fa.append_kv_cache(k, k, cache.k, cache.v, cache.table, cache.lengths([1]))
    assert cache.k._version > was


# ------------------------------------------------------------------------------------------------ decode
def check_decode(held, page, heads, kv_heads, d, dtype, layout="slots", scale=None, spread=1.0, seed=5):
    cache = Cache(held, held, page, kv_heads, d, dtype, seed, layout, spread=spread)
    q = normal(len(held), heads, d, dtype=dtype, seed=seed)
    out = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths(), scale)
    want, absolute, largest = exact_decode(q, cache.keys, cache.values, scale)
    off = (out.double() - want).abs()
    assert (off <= decode_tolerance(dtype, want, absolute, largest, d, max(held))).all(), off.max()
    for s, n in enumerate(held):
        if n <= 0:
            assert (out[s] == 0).all()
    again = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths(), scale)
    assert torch.equal(out, again)
    return out


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 128, 136, 192, 256])
def test_decode_head_dims(dtype, d):
    check_decode([1, 0, 63, 64, 65, 300], 16, 4, 2, d, dtype)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (5, 1), (8, 1), (9, 1), (16, 2), (32, 2), (17, 1), (40, 2), (128, 1)])
def test_decode_head_layouts(heads, kv_heads):
    check_decode([70, 1, 200], 16, heads, kv_heads, 64, BF16)
    check_decode([70, 1, 200], 16, heads, kv_heads, 128, FP16)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 100, 256])
@pytest.mark.parametrize("layout", ["slots", "heads"])
def test_decode_pages(page, layout):
    check_decode([1, 2, 3, 64, 99, 100, 101, 257], page, 4, 2, 64, BF16, layout)


@pytest.mark.parametrize("page", [1, 2, 7])
@pytest.mark.parametrize("heads,kv_heads,d,dtype", [(4, 2, 64, BF16), (3, 1, 40, FP16), (4, 2, 24, BF16), (4, 2, 128, FP16), (16, 1, 72, BF16),
                                                    (2, 2, 256, BF16), (9, 1, 200, FP16)])
def test_decode_pages_of_odd_and_small_size(page, heads, kv_heads, d, dtype):
    """Pages of odd size come in another way, whatever else is the same."""
    check_decode([1, 0, 63, 64, 65, 300], page, heads, kv_heads, d, dtype)


@pytest.mark.parametrize("held", [[1], [900], [40000], [1, 20000, 0, 3], [0, 0, 0], [5000] * 7, list(range(200)), [17] * 600])
def test_decode_lengths(held):
    check_decode(held, 16, 8, 2, 64, BF16)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (FP16, 128), (BF16, 256)])
def test_decode_long(dtype, d):
    check_decode([30000, 100, 131072 // (d // 128)], 64, 16, 2, d, dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_decode_peaked(dtype):
    """Scores of a few hundred: almost all weights vanish, and the running maximum moves often."""
    check_decode([400, 3000], 16, 4, 2, 64, dtype, scale=0.5, spread=8.0)


def test_decode_offsets_beyond_32_bits():
    """A cache of more than 2^32 elements, read at both ends."""
    pages, page, kv_heads, d = 1 << 15, 128, 8, 128
    k = torch.empty(pages, page, kv_heads, d, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() >= 1 << 32
    ends = [0, pages - 1, 1, pages - 2]
    keys, values = normal(512, kv_heads, d, dtype=BF16), normal(512, kv_heads, d, dtype=BF16, seed=2)
    table = torch.tensor([ends], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([512], dtype=torch.int32, device="cuda")
    fa.append_kv_cache(keys, values, k, v, table, lengths, cu_seqlens=cu_seqlens_of([512]))
    assert torch.equal(k[ends].flatten(0, 1), keys) and torch.equal(v[ends].flatten(0, 1), values)
    q = normal(1, 16, d, dtype=BF16)
    out = fa.flash_attention_decode(q, k, v, table, lengths)
    want, absolute, largest = exact_decode(q, [keys], [values])
    assert ((out.double() - want).abs() <= decode_tolerance(BF16, want, absolute, largest, d, 512)).all()


def test_decode_infinities_and_nan():
    """Within the length they spread as the formula says; behind it, and in other sequences, they do not."""
    cache = Cache([100, 100, 100], [100] * 3, 16, 2, 64, BF16)  # everything behind is NaN
    q = normal(3, 4, 64, dtype=BF16).abs()
    clean = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    assert clean.isfinite().all()
    at = cache.places(1, [99])
    keep = cache.v[at].clone()
    cache.v[at] = math.inf
    out = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    assert torch.equal(out[[0, 2]], clean[[0, 2]]) and (out[1] == math.inf).all()
    out = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths([100, 99, 100]))
    assert out.isfinite().all()
    cache.v[at] = keep
    cache.k[cache.places(1, [3])] = -math.inf  # the scores of one key are -inf (q is positive): its weight is 0
    out = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    keys, values = [torch.cat([t[1][:3], t[1][4:]]) for t in (cache.keys, cache.values)]
    want, absolute, largest = exact_decode(q[1:2], [keys], [values])
    assert ((out[1:2].double() - want).abs() <= decode_tolerance(BF16, want, absolute, largest, 64, 100)).all()
    cache.k[cache.places(1, range(100))] = -math.inf  # no finite score: no softmax
    out = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    assert out[1].isnan().all() and torch.equal(out[[0, 2]], clean[[0, 2]])


def test_decode_leaves_out_pages_outside_the_cache():
    cache = Cache([100, 50], [100, 50], 16, 2, 64, BF16)
    q = normal(2, 4, 64, dtype=BF16)
    clean = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    table = cache.table.clone()
    table[0, 2], table[0, 5] = -5, 2**31 - 1
    out = fa.flash_attention_decode(q, cache.k, cache.v, table, cache.lengths())
    assert _lib.device_status() == 0x40002
    left = [i for i in range(100) if i // 16 not in (2, 5)]
    want, absolute, largest = exact_decode(q[:1], [cache.keys[0][left]], [cache.values[0][left]])
    assert ((out[:1].double() - want).abs() <= decode_tolerance(BF16, want, absolute, largest, 64, 100)).all()
    assert torch.equal(out[1], clean[1])


def test_decode_lengths_beyond_the_table_are_cut():
    cache = Cache([112, 16], [112, 16], 16, 2, 64, BF16)
    q = normal(2, 4, 64, dtype=BF16)
    a = fa.flash_attention_decode(q[:1], cache.k, cache.v, cache.table[:1], cache.lengths([112]))
    b = fa.flash_attention_decode(q[:1], cache.k, cache.v, cache.table[:1], cache.lengths([2**31 - 1]))
    assert torch.equal(a, b)
    assert (fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths([-(2**31), -1])) == 0).all()


def test_decode_strided_inputs():
    cache = Cache([90, 33], [90, 33], 16, 2, 64, BF16)
    fused = normal(2, 8, 64, dtype=BF16)
    q = fused[:, 2:6]
    wide = torch.zeros(2, 32, dtype=torch.int32, device="cuda")
    wide[:, 5 : 5 + cache.table.shape[1]] = cache.table
    a = fa.flash_attention_decode(q, cache.k, cache.v, wide[:, 5 : 5 + cache.table.shape[1]], cache.lengths())
    b = fa.flash_attention_decode(q.contiguous(), cache.k, cache.v, cache.table, cache.lengths())
    assert torch.equal(a, b)
    both = torch.stack([cache.k, cache.v], 1)  # [pages, 2, page, heads, d]
    c = fa.flash_attention_decode(q, both[:, 0], both[:, 1], cache.table, cache.lengths())
    assert torch.equal(c, b)
    same = cache.table[:1].expand(2, -1)  # two sequences of one table row
    d = fa.flash_attention_decode(q, cache.k, cache.v, same, cache.lengths([90, 90]))
    assert torch.equal(d[0], b[0])


def test_decode_on_another_stream_and_captured():
    cache = Cache([200, 90, 0], [260, 260, 260], 16, 2, 128, BF16)
    q, k, v = (normal(3, h, 128, dtype=BF16, seed=s) for s, h in ((1, 8), (2, 2), (3, 2)))
    cos, sin = fa.rotary_tables(300, 128, device="cuda")
    lengths = cache.lengths()

    def step():
        lengths.add_(lengths > 0)
        turned, _ = fa.append_kv_cache(k, v, cache.k, cache.v, cache.table, lengths, q=q, cos=cos, sin=sin)
        return fa.flash_attention_decode(turned, cache.k, cache.v, cache.table, lengths)

    start = cache.k.clone(), cache.v.clone(), lengths.clone()
    want = [step().clone() for _ in range(6)]
    for now, was in zip((cache.k, cache.v, lengths), start):
        now.copy_(was)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step() for _ in range(2)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # a captured step is not run
        out = step()
    for i in range(2, 6):
        graph.replay()
        assert torch.equal(out, want[i])


def test_two_captured_steps_replayed_at_the_same_time():
    """Each graph has a workspace of its own."""
    caches = [Cache([5000, 100], [5000, 100], 16, 2, 64, BF16, seed=s) for s in (1, 2)]
    q = normal(2, 16, 64, dtype=BF16)
    want = [fa.flash_attention_decode(q, c.k, c.v, c.table, c.lengths()) for c in caches]
    graphs, outs, lengths = [], [], [c.lengths() for c in caches]
    for c, n in zip(caches, lengths):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fa.flash_attention_decode(q, c.k, c.v, c.table, n))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_status_check_raises(monkeypatch):
    cache = Cache([40], [40], 16, 2, 64, BF16)
    q = normal(1, 4, 64, dtype=BF16)
    monkeypatch.setenv("FA2_B200_CHECK_STATUS", "1")
    fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    with pytest.raises(_lib.Fa2Error, match="outside the cache"):
        fa.flash_attention_decode(q, cache.k, cache.v, torch.full_like(cache.table, -1), cache.lengths())


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_decode_on_the_other_device():
    cache = Cache([100], [100], 16, 2, 64, BF16)
    q = normal(1, 4, 64, dtype=BF16)
    want = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    out = fa.flash_attention_decode(*(t.to("cuda:1") for t in (q, cache.k, cache.v, cache.table, cache.lengths())))
    assert torch.equal(out.cpu(), want.cpu())


@pytest.mark.parametrize("where", [0, 63, 64, 2999])
def test_decode_nan_reaches_the_output(where):
    """A NaN key stays visible wherever its 16 keys end up among the parts that are joined, alone in them too."""
    cache = Cache([3000, 65], [3000, 65], 16, 2, 64, BF16)
    q = normal(2, 4, 64, dtype=BF16)
    clean = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    cache.k[cache.places(0, [where])] = math.nan
    cache.k[cache.places(1, [64])] = math.nan  # the only key of its 16
    out = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    assert clean.isfinite().all() and out.isnan().all()
