"""Packed documents on the host: workspace sizes, refusals of the C entries (checked before any launch), frequencies
and the oracle itself (no GPU)."""
import re

import numpy as np
import pytest
import torch

from mme import _lib, ops
from oracle import docs as oracle


def ws(n, rows, keys, Hq, Hkv, hd, max_rows):
    return _lib.query("mme_attention_docs_workspace_bytes", n, rows, keys, Hq, Hkv, hd, max_rows)


@pytest.mark.parametrize("args", [(0, 0, 0, 1, 1, 64, 0), (1, 0, 5000, 8, 1, 256, 0), (3, 10, 0, 8, 1, 256, 10),
                                  (3, 10, 90000, 8, 1, 256, 0), (1, 2147483647, 2147418111, 1, 1, 8, 2147483647),
                                  (2147483646, 1, 1, 65535, 65535, 256, 1), (100000, 100000, 2000000000, 64, 64, 128, 1)])
def test_workspace_sizes_of_the_ends(args):
    assert ws(*args) >= 0


def test_workspace_is_for_few_rows_and_many_keys_alone():
    assert ws(1, 1, 60000, 8, 1, 256, 1) > 0
    assert ws(1, 60000, 60000, 8, 1, 256, 60000) == 0        # as many rows as keys
    assert ws(64, 64, 64 * 100, 8, 1, 256, 1) == 0           # short documents
    assert ws(1, 1, 60000, 8, 1, 12, 1) == 0                 # refused
    # chunks of at least a tile for two rounds of workgroups: some ten thousand partial rows at most
    assert ws(64, 64, 64 * 100000, 32, 8, 128, 1) < 64 << 20


def test_workspace_is_none_where_the_header_says_so():
    r = np.random.RandomState(3)
    some = 0
    for _ in range(3000):
        n, hkv, group = int(r.randint(1, 300)), int(r.choice([1, 2, 8, 16])), int(r.choice([1, 2, 4, 8]))
        hd = int(r.choice([8, 64, 72, 80, 128, 192, 256]))
        keys, rows = int(n * 2 ** r.uniform(0, 16)), int(n * 2 ** r.uniform(0, 8))
        most = int(2 ** r.uniform(0, 10))
        size = ws(n, rows, keys, hkv * group, hkv, hd, most)
        some += size > 0
        assert size == 0 or (min(most, rows) * group <= 256 and keys * hd >= 40960 * n)
    assert some > 100


DOCS = dict(q=16, ldq=512, k=16, ldk=128, v=16, ldv=128, out=16, ldo=512, q_off=16, k_off=16, n=2, rows_q=8, rows_k=8, Hq=8,
            Hkv=2, hd=64, max_rows=8, causal=1, prefix=None, softcap=0.0, slopes=None, scale=0.1, ws=None, ws_bytes=0)


@pytest.mark.parametrize("change,match", [
    (dict(hd=12), "head_dim 12"), (dict(hd=136), "head_dim 136"), (dict(hd=512), "head_dim 512"), (dict(Hkv=3), "8 heads over 3"),
    (dict(Hkv=0), "over 0"), (dict(n=-1), "bad shape"), (dict(max_rows=-1), "bad shape"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(softcap=-1.0), "softcap"), (dict(softcap=2e3), "softcap"),
    (dict(softcap=float("nan")), "softcap"), (dict(causal=0, prefix=16), "prefix"), (dict(q=None), "null"),
    (dict(v=None), "null"), (dict(k_off=None), "null"), (dict(ldq=511), "leading"), (dict(ldk=127), "leading"),
    (dict(ldo=504), "leading"), (dict(ldv=1 << 24), "2\\^24"), (dict(q=8), "misaligned"), (dict(out=24), "misaligned"),
    (dict(q_off=18), "misaligned"), (dict(rows_k=2147483647), "too many"),
    (dict(n=20000000, Hq=16, Hkv=16, ldq=1024, ldk=1024, ldv=1024, ldo=1024), "too many"),
    (dict(rows_q=2147483647, max_rows=2147483647), "too many"),
    (dict(n=1, rows_q=1, rows_k=60000, max_rows=1), "workspace"),
    (dict(n=1, rows_q=1, rows_k=60000, max_rows=1, ws=16, ws_bytes=100), "workspace"),
    (dict(n=1, rows_q=1, rows_k=60000, max_rows=1, ws=8, ws_bytes=1 << 40), "workspace")])
def test_attention_docs_refusals(change, match):
    with pytest.raises(_lib.MMEError, match=match):
        _lib.call("mme_attention_docs", *{**DOCS, **change}.values(), None)


ROPE = dict(x=16, ldx=128, y=16, ldy=128, rows=4, nheads=2, hd=64, pairs=32, pos=16, ldp=4, naxes=1, freqs=16, axes=16,
            adjacent=0, inverse=0)


@pytest.mark.parametrize("change,match", [
    (dict(pairs=33), "33 pairs"), (dict(pairs=0), "0 pairs"), (dict(nheads=0), "bad shape"), (dict(rows=-1), "bad shape"),
    (dict(naxes=0), "bad shape"), (dict(ldx=127), "leading"), (dict(ldp=-1), "leading"), (dict(ldy=130), "in place"),
    (dict(x=None), "null"), (dict(freqs=None), "null"), (dict(freqs=12), "misaligned"), (dict(x=17), "misaligned"),
    (dict(nheads=65535, hd=4096, ldx=1 << 40, ldy=1 << 40), "rows of"),
    (dict(rows=2147483647, hd=4096, pairs=2048, ldx=8192, ldy=8192, ldp=2147483647), "too many"),
    (dict(rows=2147483647, hd=2048, pairs=1024, ldx=4096, ldy=4096, ldp=2147483647), "too many")])
def test_rope_axes_refusals(change, match):
    with pytest.raises(_lib.MMEError, match=match):
        _lib.call("mme_rope_axes", *{**ROPE, **change}.values(), None)


def test_no_work_is_no_error():
    _lib.call("mme_rope_axes", *{**ROPE, "rows": 0, "x": None, "y": None, "pos": None}.values(), None)
    for change in (dict(n=0), dict(rows_q=0, q=None), dict(max_rows=0)):
        _lib.call("mme_attention_docs", *{**DOCS, **change}.values(), None)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    off = torch.tensor([0, 4], dtype=torch.int32)
    f, a = ops.rope_axes_freqs((32,), 1e4, device="cpu")
    with pytest.raises(ValueError, match="CPU tensor"):
        ops.attention_docs(x, x, x, off, 2, 2)
    with pytest.raises(ValueError, match="CPU tensor"):
        ops.rope_axes(x, torch.zeros(1, 4, dtype=torch.int32), f, a, 2)


def test_rope_axes_freqs():
    f, a = ops.rope_axes_freqs((2, 3), 100.0, device="cpu")
    assert a.tolist() == [0, 0, 1, 1, 1] and a.dtype == torch.int32 and f.dtype == torch.float64
    assert torch.allclose(f, 100.0 ** (-torch.arange(5).double() / 5), rtol=1e-15)
    f, a = ops.rope_axes_freqs((2, 0, 3), 100.0, in_turns=True, per_axis=True, device="cpu")
    assert a.tolist() == [0, 2, 0, 2, 2]
    assert torch.allclose(f, torch.tensor([1.0, 1.0, 0.1, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)], dtype=torch.float64), rtol=1e-15)


def test_the_oracle_against_torch():
    """One document without a mask is torch's softmax attention in float64; the rotation is a complex product."""
    r = np.random.RandomState(0)
    q, k, v = r.randn(7, 32), r.randn(9, 16), r.randn(9, 16)
    o, _, _ = oracle.attention_docs(q, k, v, [0, 7], 4, 2, key_offsets=[0, 9])
    t = lambda x, h: torch.from_numpy(x).view(x.shape[0], h, 8).transpose(0, 1)  # noqa: E731
    kk, vv = t(k, 2).repeat_interleave(2, 0), t(v, 2).repeat_interleave(2, 0)
    want = torch.softmax(t(q, 4) @ kk.transpose(1, 2) / 8 ** 0.5, -1) @ vv
    assert np.allclose(o, want.transpose(0, 1).reshape(7, 32).numpy(), atol=1e-14)
    o, _, _ = oracle.attention_docs(q, k, v, [0, 7], 4, 2, key_offsets=[0, 9], causal=True)
    seen = torch.arange(9)[None, :] <= torch.arange(7)[:, None] + 2
    s = (t(q, 4) @ kk.transpose(1, 2) / 8 ** 0.5).masked_fill(~seen, -float("inf"))
    assert np.allclose(o, (torch.softmax(s, -1) @ vv).transpose(0, 1).reshape(7, 32).numpy(), atol=1e-14)
    x = r.randn(3, 8)
    y, _ = oracle.rope_axes(x, np.array([[1, 2, 3], [5, 7, 9]]), [1.0, 0.5], [0, 1], 2, 4, adjacent=True)
    z = (x[:, 0::2] + 1j * x[:, 1::2]) * np.exp(1j * np.array([[1.0, 2.5], [2.0, 3.5], [3.0, 4.5]]))[:, [0, 1, 0, 1]]
    assert np.allclose(y[:, 0::2], z.real, atol=1e-14) and np.allclose(y[:, 1::2], z.imag, atol=1e-14)


@pytest.mark.parametrize("n,rows,Hq,Hkv", [(1 << 30, 1, 4, 4), (1 << 28, 1 << 28, 16, 16), (1 << 30, 1 << 30, 8, 4),
                                           (1 << 30, 1, 8, 8), (2147483647, 2147483647, 65535, 65535)])
def test_products_of_documents_and_key_heads_past_32_bits(n, rows, Hq, Hkv):
    """A product that is a multiple of 2^32 was a division by zero: the sizes are answered, the call is refused."""
    assert ws(n, rows, rows, Hq, Hkv, 64, 1) == 0
    wide = dict(ldq=Hq * 64, ldk=Hkv * 64, ldv=Hkv * 64, ldo=Hq * 64)
    with pytest.raises(_lib.MMEError, match="too many"):
        _lib.call("mme_attention_docs", *{**DOCS, **wide, "n": n, "rows_q": rows, "rows_k": rows, "Hq": Hq, "Hkv": Hkv,
                                          "max_rows": 1}.values(), None)


class OnDevice(torch.Tensor):
    """A CPU tensor that says it lies on device 0: the wrappers' own checks run without a GPU."""

    def get_device(self):
        return 0


@pytest.fixture
def no_launch(monkeypatch):
    calls = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "call", lambda *args: calls.append(args))
    return calls


def here(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)


def test_rope_axes_heads_that_do_not_divide_a_row(no_launch):
    """9 heads of 72 and 16 more columns are not 9 heads of 73; with hd given they are what they are."""
    f, a = (t.as_subclass(OnDevice) for t in ops.rope_axes_freqs((18, 18), 1e4, device="cpu"))
    x, pos = here(4, 9 * 72 + 16), here(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="9 heads"):
        ops.rope_axes(x, pos, f, a, 9)
    assert not no_launch
    assert ops.rope_axes(x, pos, f, a, 9, hd=72).shape == (4, 648)
    assert ops.rope_axes(x[:, :648], pos, f, a, 9).shape == (4, 648)
    assert [c[7] for c in no_launch] == [72, 72]


AT = 1 << 20


@pytest.mark.parametrize("change", [
    dict(q=AT), dict(k=AT), dict(v=AT), dict(q=AT + 7 * 1024 + 1008), dict(v=AT - 7 * 256 - 112, ldv=128),
    dict(q=AT + 1008, ldo=1024, ldq=1024), dict(k=AT + 992, ldo=1024, ldk=1024), dict(k=AT - 240, ldo=1024, ldk=1024),
    dict(v=AT + 4096 - 16, ldo=1024, ldv=2048), dict(q=AT + 6 * 2048 + 1008, ldo=1024, ldq=4096)])
def test_attention_docs_refuses_an_out_over_its_inputs(change):
    """out is 8 rows of 1 024 bytes, k and v 8 of 256; what a change moves meets it by 16 bytes or more."""
    apart = dict(q=1 << 30, k=2 << 30, v=3 << 30, out=AT)
    with pytest.raises(_lib.MMEError, match="overlap"):
        _lib.call("mme_attention_docs", *{**DOCS, **apart, **change}.values(), None)


@pytest.mark.parametrize("change", [dict(y=AT + 2), dict(y=AT - 254), dict(y=AT + 256 * 3 + 254), dict(y=AT + 254, ldx=256, ldy=256),
                                    dict(y=AT + 2 * 256 + 16, ldx=256, ldy=384)])
def test_rope_axes_refuses_rows_that_overlap(change):
    """4 rows of 256 bytes, turned into rows that share some but not all of their places with them."""
    with pytest.raises(_lib.MMEError, match="overlap"):
        _lib.call("mme_rope_axes", *{**ROPE, "x": AT, **change}.values(), None)


@pytest.mark.parametrize("change", [dict(scale=3e38), dict(scale=1e36, softcap=1e-3), dict(scale=1.2e38, softcap=1.0)])
def test_scales_whose_products_leave_32_bits_are_refused(change):
    """scale log2(e), or 2 log2(e) scale / softcap, infinite in fp32: a score of 0 would come out as 0 x infinity."""
    with pytest.raises(_lib.MMEError, match="scale"):
        _lib.call("mme_attention_docs", *{**DOCS, "out": 1 << 20, "q": 1 << 21, "k": 1 << 22, "v": 1 << 23, **change}.values(), None)


def test_no_kernel_that_nothing_launches():
    """One-wave workgroups with whole keys are for head dims to 128: the wide head dims make no kernel of that form."""
    with open(_lib.LIB_PATH, "rb") as f:
        names = set(re.findall(rb"attn_docs_kernelILi(\d+)ELb([01])ELi(\d+)ELi(\d+)ELb([01])ELb([01])ELi([0-3])E", f.read()))
    assert len({n[:2] for n in names}) == 8      # five head dims of their own, three general widths
    # a head dim has the split form and the one for four waves, up to 128 the one for one wave too; four scores each
    assert len(names) == 4 * (6 * 3 + 2 * 2)
