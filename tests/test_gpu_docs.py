"""Rotary positions with several axes and attention over packed documents, against the 64-bit oracle."""
import numpy as np
import pytest
import torch

from oracle import docs as oracle

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HALF = 2.0 ** -8   # half a bf16 step, relative


def randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(BF16)


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) % (1 << 31) if len(seed) > 1 else seed[0])


# ------------------------------------------------------------------ rope_axes
def check_rope(y, x, pos, freqs, axes, nheads, hd, **kw):
    want, size = oracle.rope_axes(x.double().numpy(), pos.numpy(), freqs.numpy(), axes.numpy(), nheads, hd, **kw)
    got = y.double().cpu().numpy()[:, :nheads * hd]
    # the rounding of the result, and of the sine and cosine: the fraction of a turn in fp32 (2^-25 turns = 2^-22.3)
    # and the sine unit's own error, taken at 2^-19 in all, and three fp32 roundings of the products
    tol = HALF * np.abs(want) + (2.0 ** -19 + 3 * 2.0 ** -24) * size
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) - tol)


ROPE = [
    # rows, heads, hd, sections, theta, in_turns, per_axis, adjacent, far
    (1, 1, 64, (32,), 1e4, False, False, False, 1),
    (21, 9, 256, (32, 48, 48), 1e4, False, False, False, 1000),
    (130, 5, 72, (18, 18), 1e4, False, True, False, 64),          # 8-byte vectors
    (67, 3, 80, (10, 10, 10, 10), 1e2, True, False, True, 5000),
    (33, 24, 64, (8, 8, 8), 1e6, True, False, True, 1000000),      # three quarters of a head
    (40, 2, 72, (9, 8), 1e4, False, True, False, 300),             # single elements
    (40, 2, 30, (5, 4), 1e4, True, True, True, 300),
    (9, 3, 2, (1,), 1e4, False, False, False, 100),
    (300, 1, 128, (64,), 1e4, False, False, False, 2147483000),    # the far end of int32
    (257, 40, 64, (0, 32), 1e4, False, False, True, 100),          # an axis with no pairs; several heads a thread
    (3000, 33, 64, (16, 8), 1e4, False, False, False, 100),
]


@pytest.mark.parametrize("case", ROPE, ids=lambda c: "x".join(map(str, c[:3])))
@pytest.mark.parametrize("inverse", [False, True])
def test_rope_axes(cuda, case, inverse):
    from mme import ops
    rows, heads, hd, sections, theta, turns, per_axis, adjacent, far = case
    g = gen(rows * 7 + hd)
    x = randn(g, rows, heads * hd)
    pos = torch.randint(-far // 2, far, (len(sections), rows), generator=g, dtype=torch.int64).to(torch.int32)
    freqs, axes = ops.rope_axes_freqs(sections, theta, in_turns=turns, per_axis=per_axis, device=cuda)
    args = (pos.to(cuda), freqs, axes, heads)
    y = ops.rope_axes(x.to(cuda), *args, adjacent=adjacent, inverse=inverse)
    few = slice(0, 200)
    check_rope(y[few], x[few], pos[:, few], freqs.cpu(), axes.cpu(), heads, hd, adjacent=adjacent, inverse=inverse)
    z = x.to(cuda)
    assert ops.rope_axes(z, *args, adjacent=adjacent, inverse=inverse, out=z) is z
    assert torch.equal(z, y)


def test_rope_axes_strides_and_what_it_leaves(cuda):
    """Views of packed q | k | v rows: the first heads turn, the rest and the rows' other columns stay."""
    from mme import ops
    g = gen(3)
    x = randn(g, 50, 9 * 72 + 16).to(cuda)
    pos = torch.randint(0, 99, (2, 64), generator=g).to(torch.int32).to(cuda)[:, :50]
    freqs, axes = ops.rope_axes_freqs((18, 18), 1e4, per_axis=True, device=cuda)
    keep = x.clone()
    out = torch.full((50, 10 * 72), 7.0, dtype=BF16, device=cuda)
    ops.rope_axes(x, pos, freqs, axes, 5, hd=72, out=out)
    assert torch.equal(x, keep) and (out[:, 5 * 72:] == 7).all()
    check_rope(out, x.cpu(), pos.cpu(), freqs.cpu(), axes.cpu(), 5, 72)
    ops.rope_axes(x, pos, freqs, axes, 5, hd=72, out=x)
    assert torch.equal(x[:, :360], out[:, :360]) and torch.equal(x[:, 360:], keep[:, 360:])
    # odd leading dims and a base off 16 bytes
    odd = randn(g, 20, 2 * 64 + 3).to(cuda)[:, 1:]
    f1, a1 = ops.rope_axes_freqs((32,), 1e4, device=cuda)
    p1 = torch.arange(20, dtype=torch.int32, device=cuda)[None]
    check_rope(ops.rope_axes(odd, p1, f1, a1, 2, hd=64), odd.cpu(), p1.cpu(), f1.cpu(), a1.cpu(), 2, 64)
    # 4-byte alignment, both layouts, in and out of place
    four = randn(g, 20, 2 * 64 + 2).to(cuda)[:, 2:]
    for adjacent in (False, True):
        want = ops.rope_axes(four, p1, f1, a1, 2, hd=64, adjacent=adjacent)
        check_rope(want, four.cpu(), p1.cpu(), f1.cpu(), a1.cpu(), 2, 64, adjacent=adjacent)
        inside = torch.empty(20, 130, dtype=BF16, device=cuda)[:, 2:].copy_(four)
        assert torch.equal(ops.rope_axes(inside, p1, f1, a1, 2, hd=64, adjacent=adjacent, out=inside), want)
    # one row of positions for all axes
    f3, a3 = ops.rope_axes_freqs((10, 11, 11), 1e4, device=cuda)
    assert torch.equal(ops.rope_axes(odd, p1.expand(3, 20), f3, a3, 2, hd=64), ops.rope_axes(odd, p1, f1, a1, 2, hd=64))
    # axes outside the positions are clamped, no rows are no work
    a2 = torch.full_like(a1, 5)
    assert torch.equal(ops.rope_axes(odd, p1, f1, a2, 2, hd=64), ops.rope_axes(odd, p1, f1, a1, 2, hd=64))
    assert ops.rope_axes(odd[:0], p1[:, :0], f1, a1, 2, hd=64).shape == (0, 128)


@pytest.mark.parametrize("heads,hd,sections,adjacent", [(9, 128, (20, 22, 22), False), (32, 72, (18, 18), False),
                                                        (24, 64, (8, 8, 8), True), (6, 256, (64,), False)])
def test_rope_axes_large(cuda, heads, hd, sections, adjacent):
    """Outputs past 16 MB (streamed past the L2): rows at both ends and in the middle, and the whole against in place."""
    from mme import ops
    g = gen(hd)
    rows = 20001
    x = randn(g, rows, heads * hd)
    pos = torch.randint(0, 5000, (len(sections), rows), generator=g, dtype=torch.int64).to(torch.int32)
    freqs, axes = ops.rope_axes_freqs(sections, 1e4, device=cuda)
    y = ops.rope_axes(x.to(cuda), pos.to(cuda), freqs, axes, heads, adjacent=adjacent)
    for few in (slice(0, 40), slice(9990, 10030), slice(rows - 40, rows)):
        check_rope(y[few], x[few], pos[:, few], freqs.cpu(), axes.cpu(), heads, hd, adjacent=adjacent)
    z = x.to(cuda)
    ops.rope_axes(z, pos.to(cuda), freqs, axes, heads, adjacent=adjacent, out=z)
    assert torch.equal(z, y)


def test_rope_axes_gradient_is_the_inverse(cuda):
    """<g, d rope(x)/dx . u> by a difference along u (the map is linear) against <rope_inverse(g), u>."""
    from mme import ops
    g = gen(5)
    x, u, w = (randn(g, 64, 4 * 64).to(cuda) for _ in range(3))
    pos = torch.randint(0, 500, (3, 64), generator=g).to(torch.int32).to(cuda)
    freqs, axes = ops.rope_axes_freqs((10, 11, 11), 1e4, device=cuda)
    along = ops.rope_axes(u, pos, freqs, axes, 4).double()
    back = ops.rope_axes(w, pos, freqs, axes, 4, inverse=True).double()
    lhs, rhs = (w.double() * along).sum(), (back * u.double()).sum()
    # each of the 2 x 16384 products is off by half a bf16 step at most
    tol = HALF * ((w.double() * along).abs().sum() + (back * u.double()).abs().sum())
    assert (lhs - rhs).abs() <= tol


def test_rope_axes_refusals(cuda):
    from mme import ops
    x = torch.zeros(4, 128, dtype=BF16, device=cuda)
    pos = torch.zeros(1, 4, dtype=torch.int32, device=cuda)
    f, a = ops.rope_axes_freqs((32,), 1e4, device=cuda)
    ops.rope_axes(x, pos, f, a, 2)
    for bad in (lambda: ops.rope_axes(x.float(), pos, f, a, 2), lambda: ops.rope_axes(x, pos.long(), f, a, 2),
                lambda: ops.rope_axes(x, pos[:, :3], f, a, 2), lambda: ops.rope_axes(x, pos, f.float(), a, 2),
                lambda: ops.rope_axes(x, pos, f, a[:5], 2), lambda: ops.rope_axes(x, pos, f, a, 3),
                lambda: ops.rope_axes(x, pos, f, a, 0), lambda: ops.rope_axes(x, pos, f, a, 2, hd=65),
                lambda: ops.rope_axes(x, pos, f, a, 2, hd=60), lambda: ops.rope_axes(x.t(), pos, f, a, 2),
                lambda: ops.rope_axes(x, pos, f, a, 2, out=x[:, :100]), lambda: ops.rope_axes(x.cpu(), pos, f, a, 2),
                lambda: ops.rope_axes_freqs((), 1e4), lambda: ops.rope_axes_freqs((-1, 2), 1e4),
                lambda: ops.rope_axes_freqs((0, 0), 1e4), lambda: ops.rope_axes_freqs((4,), 0.0)):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------ attention_docs
def cuts(lens, first=0):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]) + first, dtype=torch.int32)


def check_docs(got, q, k, v, offsets, heads, kv_heads, rows=slice(None), **kw):
    f = lambda t: None if t is None else t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()  # noqa: E731
    kw = {n: f(t) if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    want, spread, reach = oracle.attention_docs(f(q), f(k), f(v), f(offsets), heads, kv_heads, **kw)
    got = got.double().cpu().numpy()
    hd = q.shape[1] // heads
    # weights: half a bf16 step each before the products, and again where their sum is of the rounded ones; the result:
    # half a step. Scores: hd fp32 additions of terms whose sizes sum to `reach`, the scaling, bias and maximum (4
    # roundings), the tanh (3 roundings of the cap), exp2 and sums of fp32 (2^-20 takes 16 roundings).
    delta = (hd + 4) * 2.0 ** -24 * np.repeat(reach, hd, 1) + 3 * kw.get("softcap", 0.0) * 2.0 ** -23 + 2.0 ** -20
    tol = HALF * (spread + 2 * np.abs(want)) + 2 * (spread + np.abs(want)) * delta
    tol += want.shape[0] * 2.0 ** -24 * spread
    got, want, tol = got[rows], want[rows], tol[rows]
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


def make(g, rows, keys, heads, kv_heads, hd, cuda, qscale=2.0, pad=0):
    q = randn(g, rows, heads * hd + pad, scale=qscale).to(cuda)[:, :heads * hd]
    kv = randn(g, keys, 2 * kv_heads * hd + pad).to(cuda)
    return q, kv[:, :kv_heads * hd], kv[:, kv_heads * hd:2 * kv_heads * hd]


HEADS = [(1, 1, 64), (4, 4, 72), (8, 1, 256), (6, 2, 80), (4, 1, 128), (3, 3, 8), (2, 1, 40), (5, 5, 96), (7, 1, 120),
         (2, 2, 144), (3, 1, 208)]
LENS = [(1,), (33, 1, 64, 0, 65, 128), (5, 77, 12, 31, 32), (0, 0, 300), (129, 2)]


@pytest.mark.parametrize("heads,kv_heads,hd", HEADS)
@pytest.mark.parametrize("lens", LENS, ids=lambda t: "_".join(map(str, t)))
@pytest.mark.parametrize("mask", ["all", "causal", "prefix"])
def test_docs_masks_and_widths(cuda, heads, kv_heads, hd, lens, mask):
    from mme import ops
    g = gen(hd * 31 + sum(lens))
    q, k, v = make(g, sum(lens), sum(lens), heads, kv_heads, hd, cuda)
    off = cuts(lens).to(cuda)
    kw = dict(causal=mask != "all")
    if mask == "prefix":
        kw["prefix"] = torch.tensor([(3 * n) // 4 if i % 3 else n + 5 if i else 0 for i, n in enumerate(lens)],
                                    dtype=torch.int32, device=cuda)
    got = ops.attention_docs(q, k, v, off, heads, kv_heads, **kw)
    check_docs(got, q, k, v, off, heads, kv_heads, **kw)


@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 4, 64), (8, 1, 256), (4, 2, 128), (3, 3, 72)])
@pytest.mark.parametrize("cap,bias,scale", [(50.0, False, None), (5.0, False, 1.0), (0.0, True, None), (30.0, True, 0.3),
                                            (0.0, False, 4.0)])
@pytest.mark.parametrize("causal", [False, True])
def test_docs_scores(cuda, heads, kv_heads, hd, cap, bias, scale, causal):
    from mme import ops
    lens = (70, 3, 200, 64)
    g = gen(hd + int(cap))
    q, k, v = make(g, sum(lens), sum(lens), heads, kv_heads, hd, cuda)
    off = cuts(lens).to(cuda)
    kw = dict(causal=causal, softcap=cap, scale=scale,
              slopes=(2.0 ** -torch.arange(1, heads + 1).float()).to(cuda) if bias else None)
    check_docs(ops.attention_docs(q, k, v, off, heads, kv_heads, **kw), q, k, v, off, heads, kv_heads, **kw)


@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 1, 256), (4, 4, 72), (8, 2, 128), (1, 1, 64)])
@pytest.mark.parametrize("klens", [(1030,), (5000, 1, 0, 777, 64, 2050), (129,) * 9])
@pytest.mark.parametrize("qlen", [1, 3])
@pytest.mark.parametrize("full", [False, True])
def test_docs_few_queries(cuda, heads, kv_heads, hd, klens, qlen, full):
    """Few rows against many keys, split and joined: documents without keys, fewer keys than queries, chunks that
    causal rows do not reach."""
    from mme import ops
    g = gen(hd + qlen + len(klens))
    n = len(klens)
    qlens = [qlen if i != 2 else 0 if qlen > 1 else 1 for i in range(n)]
    q, k, v = make(g, sum(qlens), sum(klens), heads, kv_heads, hd, cuda)
    off, koff = cuts(qlens).to(cuda), cuts(klens).to(cuda)
    kw = dict(key_offsets=koff, max_rows=qlen)
    if full:
        kw.update(causal=True, softcap=30.0, slopes=(2.0 ** -torch.arange(4, heads + 4).float()).to(cuda),
                  prefix=torch.tensor([i * 3 for i in range(n)], dtype=torch.int32, device=cuda))
    got = ops.attention_docs(q, k, v, off, heads, kv_heads, **kw)
    check_docs(got, q, k, v, off, heads, kv_heads, **kw)
    # without the promise the rows take the other way, to the same values
    kw.pop("max_rows")
    check_docs(ops.attention_docs(q, k, v, off, heads, kv_heads, **kw), q, k, v, off, heads, kv_heads, **kw)


@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 1, 40), (3, 1, 96), (2, 2, 144), (8, 1, 256), (4, 4, 72), (2, 1, 80),
                                               (8, 2, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_docs_several_blocks_of_rows_against_split_keys(cuda, heads, kv_heads, hd, causal):
    from mme import ops
    g = gen(hd * 3 + heads)
    qlens, klens = (30, 1, 17), (900, 1300, 20)
    q, k, v = make(g, sum(qlens), sum(klens), heads, kv_heads, hd, cuda)
    off, koff = cuts(qlens).to(cuda), cuts(klens).to(cuda)
    kw = dict(key_offsets=koff, max_rows=30, causal=causal)
    check_docs(ops.attention_docs(q, k, v, off, heads, kv_heads, **kw), q, k, v, off, heads, kv_heads, **kw)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_docs_masked_values_in_split_keys(cuda, value):
    """The later of two query rows sees a key whose v is not finite, the earlier one does not."""
    from mme import ops
    g = gen(23)
    q, k, v = make(g, 4, 1600, 4, 1, 128, cuda)
    off, koff = cuts((2, 2)).to(cuda), cuts((800, 800)).to(cuda)
    v[799] = value
    kw = dict(key_offsets=koff, max_rows=2, causal=True)
    got = ops.attention_docs(q, k, v, off, 4, 1, **kw)
    check_docs(got, q, k, v, off, 4, 1, rows=np.array([True, False, True, True]), **kw)
    assert not torch.isfinite(got[1].float()).any()


LARGE = [
    # document lengths, heads, kv_heads, hd, what else: enough workgroups that the longest documents go first
    ((700, 64, 1500, 0, 333, 1, 64, 900), 16, 16, 72, {}),
    ((1040, 1060, 1031), 8, 1, 256, dict(causal=True, prefix=True, softcap=50.0)),
    ((2500, 3, 1700), 16, 8, 128, dict(causal=True)),
    ((5, 40, 1900, 77, 800), 24, 24, 64, dict(slopes=True)),
    ((300,) * 40, 5, 5, 96, dict(causal=True, slopes=True, softcap=30.0)),
    ((129,) * 63, 12, 4, 80, dict(causal=True)),
    ((129,) * 64, 12, 4, 80, dict(causal=True)),
    ((2100, 1700, 1), 6, 2, 240, {}),
]


@pytest.mark.parametrize("lens,heads,kv_heads,hd,what", LARGE, ids=lambda v: str(v)[:20])
def test_docs_large(cuda, lens, heads, kv_heads, hd, what):
    """Whole outputs of large calls against float64 products on the device, a document and a head at a time."""
    from mme import ops
    g = gen(sum(lens) + hd)
    rows = sum(lens)
    q, k, v = make(g, rows, rows, heads, kv_heads, hd, cuda)
    off = cuts(lens).to(cuda)
    kw = dict(causal=what.get("causal", False), softcap=what.get("softcap", 0.0))
    if "prefix" in what:
        kw["prefix"] = torch.tensor([n * 3 // 4 for n in lens], dtype=torch.int32, device=cuda)
    if "slopes" in what:
        kw["slopes"] = (2.0 ** -torch.arange(1, heads + 1).float()).to(cuda)
    out = torch.full((rows, heads * hd), float("nan"), dtype=BF16, device=cuda)
    got = ops.attention_docs(q, k, v, off, heads, kv_heads, out=out, **kw).double()
    row = 0
    for d, n in enumerate(lens):
        at = torch.arange(n, device=cuda)
        last = at + 1
        if "prefix" in kw:
            last = torch.maximum(last, kw["prefix"][d].long())
        for h in range(heads if n else 0):
            j = h * kv_heads // heads
            qq, kk, vv = (t[row:row + n, i * hd:(i + 1) * hd].double().contiguous() for t, i in ((q, h), (k, j), (v, j)))
            s = qq @ kk.t().contiguous() * hd ** -0.5
            big = qq.abs() @ kk.abs().t().contiguous() * hd ** -0.5
            if kw["softcap"]:
                s = kw["softcap"] * torch.tanh(s / kw["softcap"])
            if "slopes" in kw:
                bias = kw["slopes"][h].double() * (at[:, None] - at[None, :]).abs()
                s, big = s - bias, big + bias
            if kw["causal"]:
                s = s.masked_fill(at[None, :] >= last[:, None], -float("inf"))
            w = torch.softmax(s, -1)
            want, spread = w @ vv, w @ vv.abs()
            # as in check_docs
            delta = (hd + 4) * 2.0 ** -24 * big.amax(1, keepdim=True) + 3 * kw["softcap"] * 2.0 ** -23 + 2.0 ** -20
            tol = HALF * (spread + 2 * want.abs()) + 2 * (spread + want.abs()) * delta + n * 2.0 ** -24 * spread
            bad = ~((got[row:row + n, h * hd:(h + 1) * hd] - want).abs() <= tol)
            assert not bad.any(), (d, h, bad.nonzero()[:5])
        row += n


def test_docs_rows_that_see_nothing_are_zero(cuda):
    from mme import ops
    g = gen(11)
    q, k, v = make(g, 90, 40, 2, 1, 64, cuda)
    off, koff = cuts((50, 40)).to(cuda), cuts((40, 0)).to(cuda)
    for max_rows in (None, 50):
        got = ops.attention_docs(q, k, v, off, 2, 1, key_offsets=koff, causal=True, max_rows=max_rows)
        check_docs(got, q, k, v, off, 2, 1, key_offsets=koff, causal=True)
        assert (got[:10] == 0).all() and (got[50:] == 0).all()
    none = ops.attention_docs(q, k[:0], v[:0], off, 2, 1, key_offsets=torch.zeros_like(off))
    assert (none == 0).all()


@pytest.mark.parametrize("split", [False, True])
def test_docs_rows_left_alone(cuda, split):
    """Rows before the first document, behind the last and past max_rows keep what they held; out may be wider."""
    from mme import ops
    g = gen(12)
    q, k, v = make(g, 30, 4000, 4, 2, 64, cuda, pad=24)
    off = torch.tensor([4, 6, 6, 11], dtype=torch.int32, device=cuda)
    koff = torch.tensor([100, 1500, 1600, 3900], dtype=torch.int32, device=cuda)
    big = torch.full((30, 4 * 64 + 8), 7.0, dtype=BF16, device=cuda)
    kw = dict(key_offsets=koff, max_rows=3, out=big[:, :256])
    assert ops.attention_docs(q, k, v, off, 4, 2, causal=not split, **kw).data_ptr() == big.data_ptr()
    before = torch.full((30, 256), 7.0)
    check_docs(big[:, :256], q, k, v, off, 4, 2, key_offsets=koff, max_rows=3, out=before, causal=not split)
    assert (big[:4] == 7).all() and (big[9:] == 7).all() and (big[:, 256:] == 7).all()


@pytest.mark.parametrize("hd", [64, 72, 128, 256])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_docs_what_masked_keys_hold_does_not_matter(cuda, hd, value):
    """Infinities and NaN in k and v: beside the documents, in another document, and at keys that some rows of a
    tile see and others do not."""
    from mme import ops
    g = gen(13)
    lens = (70, 90, 33)
    q, k, v = make(g, 200, 200, 2, 1, hd, cuda)
    off = cuts(lens, first=2).to(cuda)
    for t in (k, v):
        t[:2] = value
        t[195:] = value
        t[2 + 70 + 41] = value      # key 41 of the second document: rows from 41 on see it when causal
    bad = np.zeros(200, bool)
    bad[2 + 70 + 41:2 + 160] = True
    got = ops.attention_docs(q, k, v, off, 2, 1, causal=True)
    inside = np.zeros(200, bool)
    inside[2:195] = True
    good = torch.from_numpy(inside & ~bad).to(cuda)
    assert torch.isfinite(got[good].float()).all()
    # rows that are taken again have weights that are not rounded, which the bound of rounded ones holds as well
    check_docs(got, q, k, v, off, 2, 1, causal=True, rows=inside & ~bad)
    if value != value:
        assert torch.isnan(got[2 + 70 + 41:2 + 160].float()).all()


@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 64), (2, 2, 72), (1, 1, 96), (2, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("split", [False, True])
def test_docs_an_infinity_that_is_seen(cuda, heads, kv_heads, hd, causal, split):
    """An infinity in v at a document's last key, whose tile reaches past the document: infinite in its column for
    the rows that see it, and nowhere else."""
    from mme import ops
    g = gen(15)
    klens = (1, 33, 64, 70, 2001)
    off = cuts((1,) * 5 if split else klens).to(cuda)
    koff = cuts(klens).to(cuda)
    rows, keys = int(off[-1]), sum(klens)
    q, k, v = make(g, rows, keys, heads, kv_heads, hd, cuda)
    v[koff[1:].long() - 1, 3] = float("inf")
    got = ops.attention_docs(q, k, v, off, heads, kv_heads, key_offsets=koff, max_rows=1 if split else None, causal=causal)
    want, spread, _ = oracle.attention_docs(*(t.double().cpu().numpy() for t in (q, k, v)), off.cpu().numpy(), heads,
                                            kv_heads, key_offsets=koff.cpu().numpy(), causal=causal)
    got = got.double().cpu().numpy()
    assert np.isinf(want).sum() >= 5 and not np.isnan(want).any()
    assert np.array_equal(np.isposinf(got), np.isposinf(want)) and not np.isnan(got).any()
    # check_docs' bound is at most 3 half steps of the spread, and 2 delta < 2^-9 of it with reach < 64 and hd <= 256
    ok = np.isfinite(want)
    assert (np.abs(got[ok] - want[ok]) <= 4 * HALF * spread[ok] + 2.0 ** -20).all()


def test_docs_values_that_reach_far(cuda):
    """Scores of +-1e30, all alike, and a maximum that grows in every tile."""
    from mme import ops
    g = gen(14)
    q, k, v = make(g, 256, 256, 1, 1, 64, cuda)
    off = cuts((256,)).to(cuda)
    for f in (1e15, 0.0):
        got = ops.attention_docs((q.float() * f).to(BF16), (k.float() * max(f, 1)).to(BF16), v, off, 1, 1)
        want, _, _ = oracle.attention_docs((q.float() * f).to(BF16).double().cpu().numpy(),
                                           (k.float() * max(f, 1)).to(BF16).double().cpu().numpy(),
                                           v.double().cpu().numpy(), off.cpu().numpy(), 1, 1)
        # at 1e30 a row is its largest key's value (no two keys of these inputs tie)
        assert np.allclose(got.double().cpu().numpy(), want, rtol=4 * HALF, atol=2 * HALF)
    up = (torch.arange(256).float()[:, None] / 8).expand(256, 64).to(BF16).to(cuda)
    ones = torch.ones(256, 64, dtype=BF16, device=cuda)
    check_docs(ops.attention_docs(ones, up, v, off, 1, 1), ones, up, v, off, 1, 1)


def test_docs_many_documents(cuda):
    """5 000 documents, empty ones among them: the search for a slot's document goes several steps."""
    from mme import ops
    r = np.random.RandomState(1)
    lens = r.randint(0, 4, 5000)
    g = gen(15)
    q, k, v = make(g, int(lens.sum()), int(lens.sum()), 2, 1, 64, cuda)
    off = cuts(lens).to(cuda)
    check_docs(ops.attention_docs(q, k, v, off, 2, 1, causal=True), q, k, v, off, 2, 1, causal=True)
    klens = r.randint(200, 500, 300)
    q, k, v = make(g, 300, int(klens.sum()), 2, 2, 64, cuda)
    off, koff = cuts([1] * 300).to(cuda), cuts(klens).to(cuda)
    got = ops.attention_docs(q, k, v, off, 2, 2, key_offsets=koff, max_rows=1)
    check_docs(got, q, k, v, off, 2, 2, key_offsets=koff)


def test_docs_far_into_a_long_cache(cuda):
    """Keys whose elements lie past 2^31 and 2^32 from the cache's begin."""
    from mme import ops
    rows, ld = 540000, 8192   # 4.4e9 elements, 8.8 GB
    cache = torch.zeros(rows, ld, dtype=BF16, device=cuda)
    koff = torch.tensor([263000, 264000, 539200, 540000], dtype=torch.int32, device=cuda)
    g = gen(16)
    for a, b in ((263000, 264000), (539200, 540000)):
        cache[a:b, :256] = randn(g, b - a, 256).to(cuda)
    off = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=cuda)
    q = randn(g, 5, 4 * 64).to(cuda)
    k, v = cache[:, :128], cache[:, 128:256]
    got = ops.attention_docs(q, k, v, off, 4, 2, key_offsets=koff, max_rows=3)
    wide = ops.attention_docs(q, k, v, off, 4, 2, key_offsets=koff)
    part = torch.cat([cache[263000:264000, :256], cache[539200:540000, :256]])
    less = torch.tensor([0, 1000, 1000, 1800], dtype=torch.int32)
    for out in (got, wide):
        check_docs(out, q, part[:, :128], part[:, 128:], off, 4, 2, key_offsets=less)


def test_docs_wrong_offsets_stay_inside(cuda):
    """Offsets past the rows, negative or falling are clamped: rows come out wrong, nothing else is touched."""
    from mme import ops
    g = gen(17)
    q, k, v = make(g, 64, 600, 2, 1, 64, cuda)
    out = torch.full((66, 128), 7.0, dtype=BF16, device=cuda)
    for off, koff in (([-5, 20, 1000], [0, 700, 2000000000]), ([40, 10, 64], [600, 3, 100]),
                      ([0, 64, 64], [-2147483648, 2147483647, 5])):
        for max_rows in (None, 4):
            ops.attention_docs(q, k, v, torch.tensor(off, dtype=torch.int32, device=cuda), 2, 1, max_rows=max_rows,
                               key_offsets=torch.tensor(koff, dtype=torch.int32, device=cuda), out=out[1:65])
    torch.cuda.synchronize()
    assert (out[0] == 7).all() and (out[65] == 7).all()


def test_docs_refusals(cuda):
    from mme import _lib, ops
    q = torch.zeros(10, 4 * 64, dtype=BF16, device=cuda)
    k = torch.zeros(10, 2 * 64, dtype=BF16, device=cuda)
    off = torch.tensor([0, 10], dtype=torch.int32, device=cuda)
    pre = torch.zeros(1, dtype=torch.int32, device=cuda)
    slopes = torch.zeros(4, device=cuda)
    ok = ops.attention_docs(q, k, k, off, 4, 2, causal=True, prefix=pre, slopes=slopes, softcap=1.0)
    assert (ok == 0).all()
    assert ops.attention_docs(q, k, k, off[:1], 4, 2).shape == q.shape       # no document
    assert ops.attention_docs(q[:0], k, k, off * 0, 4, 2).shape == (0, 256)
    f = ops.attention_docs
    for bad in (lambda: f(q.float(), k, k, off, 4, 2), lambda: f(q, k, k.half(), off, 4, 2),
                lambda: f(q, k, k[:5], off, 4, 2), lambda: f(q, k, k, off, 4, 3), lambda: f(q, k, k, off, 3, 1),
                lambda: f(q, k, k, off.long(), 4, 2), lambda: f(q, k, k, off[:0], 4, 2),
                lambda: f(q, k, k, off, 4, 2, key_offsets=off[:1]), lambda: f(q, k, k, off, 4, 2, prefix=pre),
                lambda: f(q, k, k, off, 4, 2, causal=True, prefix=pre.long()),
                lambda: f(q, k, k, off, 4, 2, causal=True, prefix=off), lambda: f(q, k, k, off, 4, 2, slopes=slopes[:2]),
                lambda: f(q, k, k, off, 4, 2, slopes=slopes.double()), lambda: f(q, k, k, off, 4, 2, max_rows=-1),
                lambda: f(q.cpu(), k, k, off, 4, 2), lambda: f(q, k.t(), k, off, 4, 2),
                lambda: f(q, k, k, off, 4, 2, out=q[:5]), lambda: f(q, k, k, off, 4, 2, out=q[:, :128]),
                lambda: f(q, k, k, off, 4, 2, out=q.float())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(q, k, k, off, 4, 2, scale=0.0), lambda: f(q, k, k, off, 4, 2, scale=float("inf")),
                lambda: f(q, k, k, off, 4, 2, scale=float("nan")), lambda: f(q, k, k, off, 4, 2, softcap=-1.0),
                lambda: f(q, k, k, off, 4, 2, softcap=1e-4), lambda: f(q, k, k, off, 4, 2, softcap=1e4),
                lambda: f(q, k, k, off, 4, 2, softcap=float("nan")),
                lambda: f(q[:, :4 * 12], k[:, :2 * 12], k[:, :2 * 12], off, 4, 2),           # head dim 12
                lambda: f(q[:, 4:4 + 4 * 56], k[:, :2 * 56], k[:, :2 * 56], off, 4, 2)):     # 8-byte base
        with pytest.raises(_lib.MMEError):
            bad()


# ------------------------------------------------------------------ as they are used
def test_graph_streams_and_two_graphs(cuda):
    """Captured and replayed, on another stream, and two graphs of the split form that run one after the other."""
    from mme import ops
    g = gen(18)
    q, k, v = make(g, 6, 6000, 8, 1, 128, cuda)
    off = cuts([1] * 6).to(cuda)
    koffs = [cuts(t).to(cuda) for t in ((1000,) * 6, (10, 3000, 5, 2000, 900, 85))]
    eager = [ops.attention_docs(q, k, v, off, 8, 1, key_offsets=t, max_rows=1, causal=True, softcap=20.0) for t in koffs]
    graphs, outs = [], []
    for t in koffs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.attention_docs(q, k, v, off, 8, 1, key_offsets=t, max_rows=1, causal=True, softcap=20.0))
        graphs.append(graph)
    for _ in range(4):
        for o in outs:
            o.zero_()
        for graph in graphs:
            graph.replay()
        junk = torch.randn(1000, 1000, device=cuda) @ torch.randn(1000, 1000, device=cuda)
        torch.cuda.synchronize()
        assert junk.numel() and all(torch.equal(a, b) for a, b in zip(outs, eager))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [ops.attention_docs(q, k, v, off, 8, 1, key_offsets=t, max_rows=1, causal=True, softcap=20.0) for t in koffs]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(there, eager))


def test_a_decoder_step_over_packed_pages(cuda):
    """q | k | v product, rotation of the q and k heads by (time, height, width), attention within each page with an
    image prefix, output product; then a new token a page against the rotated keys kept from before."""
    from mme import ops
    H, hd, d = 8, 256, 512
    pages = [(4, 6, 5), (3, 3, 8), (1, 1, 1)]  # image grid h, w, and text tokens
    g = gen(19)
    pos, lens, prefix = [], [], []
    for h, w, text in pages:
        grid = torch.stack([torch.zeros(h * w), torch.arange(h * w) // w, torch.arange(h * w) % w])
        words = (torch.arange(text) + max(h, w)).expand(3, text)
        pos.append(torch.cat([grid, words], 1))
        lens.append(h * w + text)
        prefix.append(h * w)
    pos = torch.cat(pos, 1).to(torch.int32).contiguous()
    x = randn(g, sum(lens), d)
    wqkv, wo = randn(g, (H + 2) * hd, d, scale=d ** -0.5), randn(g, d, H * hd, scale=(H * hd) ** -0.5)
    freqs, axes = ops.rope_axes_freqs((32, 48, 48), 1e4, device=cuda)
    off, pre = cuts(lens).to(cuda), torch.tensor(prefix, dtype=torch.int32, device=cuda)
    qkv = ops.gemm(x.to(cuda), wqkv.to(cuda))
    plain = qkv.clone()
    ops.rope_axes(qkv, pos.to(cuda), freqs, axes, H + 1, hd=hd, out=qkv)
    check_rope(qkv, plain.cpu(), pos, freqs.cpu(), axes.cpu(), H + 1, hd)
    assert torch.equal(qkv[:, (H + 1) * hd:], plain[:, (H + 1) * hd:])
    q, k, v = qkv[:, :H * hd], qkv[:, H * hd:(H + 1) * hd], qkv[:, (H + 1) * hd:]
    kw = dict(causal=True, prefix=pre, softcap=50.0)
    o = ops.attention_docs(q, k, v, off, H, 1, **kw)
    check_docs(o, q, k, v, off, H, 1, **kw)
    y = ops.gemm(o, wo.to(cuda))
    want = o.double().cpu() @ wo.double().t()
    size = o.double().cpu().abs() @ wo.double().abs().t()
    assert ((y.double().cpu() - want).abs() <= HALF * want.abs() + H * hd * 2.0 ** -24 * size).all()
    # the last token of each page alone, against the page's keys
    last = (off[1:] - 1).long()
    one = cuts([1] * len(pages)).to(cuda)
    alone = ops.attention_docs(q[last].contiguous(), k, v, one, H, 1, key_offsets=off, max_rows=1, **kw)
    check_docs(alone, q[last], k, v, one, H, 1, key_offsets=off, **kw)


def test_out_beside_its_inputs_and_over_them(cuda):
    """Columns of one buffer are no overlap, at one leading dim or two; shared elements are refused before any launch."""
    from mme import _lib, ops
    g = gen(31)
    lens = (70, 33, 5)
    off = cuts(lens).to(cuda)
    buf = torch.zeros(108, 1024, dtype=BF16, device=cuda)
    buf[:, :512] = randn(g, 108, 512).to(cuda)
    q, k, v = buf[:, :256], buf[:, 256:384], buf[:, 384:512]
    keep = buf[:, :512].clone()
    want = ops.attention_docs(*(t.contiguous() for t in (q, k, v)), off, 4, 2, causal=True)
    assert torch.equal(ops.attention_docs(q, k, v, off, 4, 2, causal=True, out=buf[:, 512:768]), want)
    wide = torch.zeros(216, 512, dtype=BF16, device=cuda)   # rows of out at every other row of k
    kk = wide[:, 256:384].copy_(k.repeat_interleave(2, 0))
    two = ops.attention_docs(q, kk, kk, off, 4, 2, key_offsets=off * 2, out=wide.view(108, 1024)[:, :256])
    assert torch.equal(two, ops.attention_docs(q, kk.contiguous(), kk.contiguous(), off, 4, 2, key_offsets=off * 2))
    f, a = ops.rope_axes_freqs((32,), 1e4, device=cuda)
    pos = torch.arange(108, dtype=torch.int32, device=cuda)[None]
    assert torch.equal(ops.rope_axes(q, pos, f, a, 4, out=buf[:, 768:]), ops.rope_axes(q.contiguous(), pos, f, a, 4))
    assert torch.equal(buf[:, :512], keep)
    for bad in (lambda: ops.attention_docs(q, k, v, off, 4, 2, out=q), lambda: ops.attention_docs(q, k, v, off, 4, 2, out=buf[:, 376:632]),
                lambda: ops.rope_axes(q, pos, f, a, 4, out=buf[:, 64:320]),
                lambda: ops.rope_axes(buf[:100, :256], pos[:, :100], f, a, 4, out=buf[1:101, :256])):
        with pytest.raises(_lib.MMEError, match="overlap"):
            bad()
    assert torch.equal(buf[:, :512], keep)


def least_time(f, before, times=20):
    """The least of some calls' times in us, each behind a call of `before`."""
    took = []
    for _ in range(times):
        before()
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        took.append(a.elapsed_time(b) * 1e3)
    return min(took)


@pytest.mark.parametrize("hd,full", [(96, 128), (208, 256)])
def test_docs_time_does_not_hang_on_what_lds_held(cuda, hd, full):
    """Columns that a general head dim does not have come from LDS that nobody wrote. NaN left there by the call before
    sent every causal row through a search of v: the same result in twice the time."""
    from mme import ops
    g = gen(hd)
    off = cuts((1000,) * 4).to(cuda)
    q, k, v = make(g, 4000, 4000, 8, 8, hd, cuda)
    fill = cuts((300,) * 10).to(cuda)
    x = [torch.full((3000, 64 * full), f, dtype=BF16, device=cuda) for f in (0.0, float("nan"))]
    runs = [lambda t=t: ops.attention_docs(t, t, t, fill, 64, 64) for t in x]
    call = lambda: ops.attention_docs(q, k, v, off, 8, 8, causal=True)  # noqa: E731
    want = call()
    zeros, nans = (least_time(call, before) for before in runs)
    assert nans <= 1.4 * zeros, (zeros, nans)
    assert torch.equal(call(), want)


def test_one_row_whatever_its_stride(cuda):
    """A single row lies where it begins: a stride that leads nowhere (expanded, or odd) does not matter."""
    from mme import ops
    g = gen(37)
    one = cuts((1,)).to(cuda)
    f, a = ops.rope_axes_freqs((32,), 1e4, device=cuda)
    pos = torch.full((1, 1), 9, dtype=torch.int32, device=cuda)
    row = randn(g, 512).to(cuda)
    for x in (row[:256].expand(1, 256), torch.as_strided(row, (1, 256), (771, 1), 8), torch.as_strided(row, (1, 256), (3, 1), 256)):
        flat = x.reshape(256).clone()[None]
        k = flat[:, :128]
        want = ops.attention_docs(flat, k, k, one, 4, 2)
        kk = x[:, :128]
        assert torch.equal(ops.attention_docs(x, kk, kk, one, 4, 2), want)
        assert torch.equal(want, torch.cat([k[:, :64], k[:, :64], k[:, 64:], k[:, 64:]], 1))
        out = torch.as_strided(torch.zeros(800, dtype=BF16, device=cuda), (1, 256), (13, 1), 16)
        assert torch.equal(ops.attention_docs(x, kk, kk, one, 4, 2, out=out), want)
        turned = ops.rope_axes(flat, pos, f, a, 4)
        assert torch.equal(ops.rope_axes(x, pos, f, a, 4), turned)
        assert torch.equal(ops.rope_axes(x, pos, f, a, 4, out=out), turned)
        y = flat.clone()
        assert torch.equal(ops.rope_axes(y, pos, f, a, 2, hd=64, out=y[:, :128]), turned[:, :128])


# ------------------------------------------------------------------ forms that the tests above do not reach
def check_whole(got, q, k, v, off, koff, heads, kv_heads, adds, causal=False, prefix=None, softcap=0.0, slopes=None):
    """Whole outputs against float64 on the device, a document and a head at a time. The bound is check_docs', with
    `adds` fp32 additions in a row's sums of weights and of products."""
    hd = q.shape[1] // heads
    got, off, koff = got.double(), off.tolist(), koff.tolist()
    for d in range(len(off) - 1):
        m, n = off[d + 1] - off[d], koff[d + 1] - koff[d]
        p = torch.arange(m, device=q.device)[:, None] + n - m
        at = torch.arange(n, device=q.device)[None, :]
        seen = at >= 0 if not causal else at <= p if prefix is None else (at <= p) | (at < prefix[d])
        for h in range(heads if m else 0):
            j = h * kv_heads // heads
            qq = q[off[d]:off[d + 1], h * hd:(h + 1) * hd].double().contiguous()
            kk, vv = (t[koff[d]:koff[d + 1], j * hd:(j + 1) * hd].double().contiguous() for t in (k, v))
            s = qq @ kk.t().contiguous() * hd ** -0.5
            big = qq.abs() @ kk.abs().t().contiguous() * hd ** -0.5
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                bias = slopes[h].double() * (p - at).abs()
                s, big = s - bias, big + bias
            s = s.masked_fill(~seen, -float("inf"))
            w = torch.softmax(s, -1) if n else s
            w = w.masked_fill(~seen, 0.0)   # a row that sees nothing
            want, spread = w @ vv, w @ vv.abs()
            reach = big.masked_fill(~seen, 0.0).amax(1, keepdim=True) if n else 0.0
            delta = (hd + 4) * 2.0 ** -24 * reach + 3 * softcap * 2.0 ** -23 + 2.0 ** -20
            tol = HALF * (spread + 2 * want.abs()) + 2 * (spread + want.abs()) * delta + 2 * adds * 2.0 ** -24 * spread
            bad = ~((got[off[d]:off[d + 1], h * hd:(h + 1) * hd] - want).abs() <= tol)
            assert not bad.any(), (d, h, bad.nonzero()[:5])


def scores(mask, heads, klens, cuda):
    kw = dict(causal=mask != "all")
    if mask != "all" and "prefix" in mask:
        kw["prefix"] = torch.tensor([(n // 2, 0, n + 3)[i % 3] for i, n in enumerate(klens)], dtype=torch.int32, device=cuda)
    if "cap" in mask:
        kw["softcap"] = 30.0
    if "bias" in mask:
        kw["slopes"] = (2.0 ** -torch.arange(2, heads + 2).float()).to(cuda)
    return kw


@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 4, 8), (4, 4, 40), (6, 6, 64), (4, 4, 72), (8, 4, 72), (10, 5, 80), (5, 5, 96),
                                               (6, 6, 120), (8, 4, 128), (8, 8, 128)])
@pytest.mark.parametrize("mask", ["all", "causal", "prefix", "cap bias", "cap bias prefix"])
def test_docs_many_short_documents(cuda, heads, kv_heads, hd, mask):
    """96 documents of 1 to 128 rows: one wave a workgroup, tiles of 32 keys, up to four of them a document."""
    from mme import ops
    r = np.random.RandomState(hd)
    lens = np.concatenate([r.randint(1, 100, 88), [1, 31, 32, 33, 64, 96, 97, 128]]).tolist()
    rows = sum(lens)
    assert rows * (heads // kv_heads) <= 128 * 96 and (rows * (heads // kv_heads) // 32 + 96) * kv_heads >= 512
    g = gen(hd * 5 + heads)
    q, k, v = make(g, rows, rows, heads, kv_heads, hd, cuda)
    off = cuts(lens).to(cuda)
    kw = scores(mask, heads, lens, cuda)
    out = torch.full((rows, heads * hd), float("nan"), dtype=BF16, device=cuda)
    check_whole(ops.attention_docs(q, k, v, off, heads, kv_heads, out=out, **kw), q, k, v, off, off, heads, kv_heads, 128, **kw)
    # a few rows a document against up to 250 keys, some documents without keys
    klens = r.randint(0, 250, 96).tolist()
    qlens = r.randint(0, 40, 96).tolist()
    q, k, v = make(g, sum(qlens), sum(klens), heads, kv_heads, hd, cuda)
    off, koff = cuts(qlens).to(cuda), cuts(klens).to(cuda)
    kw = scores(mask, heads, klens, cuda)
    out = torch.full((sum(qlens), heads * hd), float("nan"), dtype=BF16, device=cuda)
    got = ops.attention_docs(q, k, v, off, heads, kv_heads, key_offsets=koff, out=out, **kw)
    check_whole(got, q, k, v, off, koff, heads, kv_heads, 250, **kw)


@pytest.mark.parametrize("heads,kv_heads,hd,klens", [(8, 1, 256, (20000,)), (1, 1, 64, (65536,)), (1, 1, 64, (16385, 7, 32768)),
                                                     (4, 1, 72, (50001,)), (2, 1, 40, (40000,))])
@pytest.mark.parametrize("mask", ["all", "cap bias prefix"])
@pytest.mark.parametrize("far", [False, True])
def test_docs_join_of_many_chunks(cuda, heads, kv_heads, hd, klens, mask, far):
    """A document in hundreds of chunks (32 keys at head dim 256, 64 below: 512 to 1 024), which the join takes 256 at a
    time; with far, a key well past the first 256 chunks has nearly all the weight."""
    from mme import ops
    g = gen(hd + sum(klens))
    n = len(klens)
    q, k, v = make(g, 3 * n, sum(klens), heads, kv_heads, hd, cuda)
    off, koff = cuts([3] * n).to(cuda), cuts(klens).to(cuda)
    if far:
        for d in range(n):
            k[int(koff[d]) + klens[d] * 4 // 5, :hd] = q[3 * d + 1, :hd] * 4
    kw = scores(mask, heads, klens, cuda)
    if "slopes" in kw:
        kw["slopes"] = kw["slopes"] / 1000
    got = ops.attention_docs(q, k, v, off, heads, kv_heads, key_offsets=koff, max_rows=3, **kw)
    check_whole(got, q, k, v, off, koff, heads, kv_heads, 64 + 1024, **kw)


@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 64), (2, 2, 72), (3, 3, 96), (4, 1, 128), (4, 1, 256), (2, 1, 208)])
@pytest.mark.parametrize("mask", ["causal prefix", "causal cap", "causal bias", "causal cap bias prefix"])
@pytest.mark.parametrize("form", ["four waves", "one wave", "split"])
def test_docs_rows_taken_again_with_every_score(cuda, heads, kv_heads, hd, mask, form):
    """Rows whose tile holds an infinity or NaN of v that they do not see, with prefixes, capped and biased scores; rows
    that see no key among them."""
    from mme import ops
    g = gen(hd + len(mask))
    few = form == "split"
    qlens = [5, 2, 7] if few else [90, 41, 20] + [30] * (160 if form == "one wave" else 0)
    klens = [1500, 900, 4] if few else [90, 60, 12] + [30] * (len(qlens) - 3)
    q, k, v = make(g, sum(qlens), sum(klens), heads, kv_heads, hd, cuda)
    off, koff = cuts(qlens).to(cuda), cuts(klens).to(cuda)
    kw = scores(mask, heads, klens, cuda)
    if "prefix" in kw:
        kw["prefix"][1:3] = torch.tensor([klens[1] - 9, 0], dtype=torch.int32, device=cuda)
    blind = np.zeros((sum(qlens), 1), bool)   # rows that do not see their document's bad key
    for d, (m, n) in enumerate(zip(qlens, klens)):
        at = n - 2
        v[int(koff[d]) + at] = (float("inf"), float("nan"), -float("inf"))[d % 3]
        pre = int(kw["prefix"][d]) if "prefix" in kw else 0
        blind[int(off[d]):int(off[d]) + m, 0] = [max(i + n - m + 1, pre) <= at for i in range(m)]
    got = ops.attention_docs(q, k, v, off, heads, kv_heads, key_offsets=koff, max_rows=max(qlens), **kw)
    assert blind.any() and torch.isfinite(got[torch.from_numpy(blind[:, 0]).to(cuda)].float()).all()
    seeing = torch.from_numpy(~blind[:, 0]).to(cuda)
    assert not torch.isfinite(got[seeing].float()).any()
    # check_docs' bound holds: the weights of a row taken again are not rounded
    check_docs(got, q, k, v, off, heads, kv_heads, rows=blind[:, 0], key_offsets=koff, **kw)
    assert (got[int(off[2]):int(off[2]) + qlens[2] - klens[2]] == 0).all() or qlens[2] <= klens[2]
