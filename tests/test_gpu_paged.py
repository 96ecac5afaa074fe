"""GPU: paged key-value cache (append, decode, prefill) against the float64 oracle.

Tolerances, derived from the arithmetic.  u = half a step of the type relative
to the value (bf16 2^-8, fp16 2^-11).
  append     fp32 throughout, one rounding: u |x| + 2e-6 (|a| + |b|); the second
             term bounds the angle's rounding to 32 bits after its reduction
             (2^-23 pi), the sine's and the norm's few 2^-24
  attention  the output's rounding u |out|, plus the weights' rounding to the
             cache's type: u sum p|v| (each weight off by at most u of itself),
             plus 2^-12 sum p|v| for the fp32 products and exponentials (scores
             off by at most 2^-13: D 2^-24 sum |q k| scale < 128 2^-24 10), plus
             for fp16 n 2^-25 max|v| (weights below 2^-14 are subnormal)
  lse        2^-13 (the scores) + 2^-20 |lse|
"""
import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _np(t):
    return t.detach().double().cpu().numpy()


class Cache:
    """Pages of random rows; every slot that no sequence holds is NaN or infinite."""

    def __init__(self, lengths, kv, dim, page, dtype, seed, layout="hnd", spare=3, pad=2):
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lengths]
        self.pages = sum(need) + spare
        width = max(need + [0]) + pad
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(lengths), width), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv, page, dim)
        self.k = torch.from_numpy(rng.normal(size=shape).astype(np.float32)).to(dtype)
        self.v = torch.from_numpy(rng.normal(size=shape).astype(np.float32)).to(dtype)
        held = np.zeros((self.pages, page), bool)
        for b, n in enumerate(lengths):
            p = np.arange(n)
            held[self.table[b, p // page], p % page] = True
        bad = torch.from_numpy(~held)[:, None, :, None].expand(shape)
        poison = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=dtype)
        poison = poison[torch.arange(self.k.numel()).reshape(shape) % 3]
        self.k = torch.where(bad, poison, self.k)
        self.v = torch.where(bad, poison, self.v)
        self.k_ref = np.where(_np(bad) > 0, 0.0, _np(self.k))
        self.v_ref = np.where(_np(bad) > 0, 0.0, _np(self.v))
        self.kd, self.vd = self.k.cuda(), self.v.cuda()
        if layout == "nhd":  # [page, row, head, dim] memory
            self.kd, self.vd = (t.transpose(1, 2).contiguous().transpose(1, 2)
                                for t in (self.kd, self.vd))
        self.lengths = np.asarray(lengths, np.int32)
        self.td = torch.from_numpy(self.table).cuda()
        self.ld = torch.from_numpy(self.lengths).cuda()


def _close(got, ref, mag, dtype, lens, vmax):
    u = U[dtype]
    tol = u * np.abs(ref) + (u + 2.0 ** -12) * mag
    if dtype is torch.float16:
        tol = tol + max(lens) * 2.0 ** -25 * vmax
    bad = ~(np.abs(_np(got) - ref) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5], np.abs(_np(got) - ref).max())


def _check(out, lse, cache, q, cu, dtype, **kw):
    dim = q.shape[-1]
    kw.setdefault("scale", dim ** -0.5)
    ref, mag, l_ref = paged.attention(_np(q), cache.k_ref, cache.v_ref, cache.table, cache.lengths,
                                      cu, **kw)
    n = cu[-1]
    _close(out[:n], ref[:n], mag[:n], dtype, list(cache.lengths) + [1], np.abs(cache.v_ref).max())
    if lse is not None:
        got, l_ref = _np(lse)[:n], l_ref[:n]
        none = np.isinf(l_ref)
        assert (got[none] == -np.inf).all()
        assert (np.abs(got[~none] - l_ref[~none])
                <= 2.0 ** -13 + 2.0 ** -20 * np.abs(l_ref[~none])).all()


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,page,hq,kv,half,inter,norm,layout", [
    (128, 16, 4, 2, 64, False, True, "hnd"), (128, 64, 3, 3, 64, True, False, "nhd"),
    (64, 32, 7, 1, 32, False, True, "nhd"), (64, 16, 1, 1, 8, True, True, "hnd"),
    (128, 128, 5, 5, 16, False, False, "hnd"), (64, 256, 16, 2, 24, False, True, "hnd"),
    (128, 16, 2, 1, 0, False, True, "hnd"), (64, 16, 2, 2, 0, False, False, "hnd")])
def test_append(cuda, dtype, dim, page, hq, kv, half, inter, norm, layout):
    from hybrid_llm_b200 import kernels
    dt = DT[dtype]
    new = [5, 0, 1, 40, 17, 3]
    lengths = [5, 9, 300, 41, 17, 0]  # the last has tokens but no positions
    cache = Cache(lengths, kv, dim, page, dt, seed=dim + page + hq, layout=layout)
    rng = np.random.default_rng(5)
    cu = np.concatenate([[0], np.cumsum(new)])
    n = cu[-1] + 4                    # rows behind the last sequence
    fused = torch.from_numpy(rng.normal(size=(n, (hq + 2 * kv) * dim)).astype(np.float32)).to(dt)
    fused = fused.cuda()
    q = fused[:, :hq * dim].view(n, hq, dim)
    k = fused[:, hq * dim:(hq + kv) * dim].view(n, kv, dim)
    v = fused[:, (hq + kv) * dim:].view(n, kv, dim)
    inv = torch.tensor(10000.0 ** (-np.arange(half) / max(half, 1)), dtype=torch.float32).cuda()
    wq, wk = (torch.from_numpy(rng.normal(1, 0.3, dim).astype(np.float32)).cuda() if norm else None
              for _ in range(2))
    q_out = torch.full((n, hq, dim), 7.0, dtype=dt, device="cuda")
    before = cache.kd.clone(), cache.vd.clone()
    got = kernels.paged_append(q, k, v, cache.kd, cache.vd, cache.td, cache.ld,
                               cu_q=torch.from_numpy(cu.astype(np.int32)).cuda(),
                               inv_freq=inv if half else None, interleaved=inter, q_norm=wq,
                               k_norm=wk, q_out=q_out)
    kernels.check_device_status()
    assert got is q_out
    seq, pos = paged.positions(cu, lengths, n)
    live = (seq >= 0) & (pos >= 0)
    args = (1e-6, pos, inv.cpu().numpy() if half else None, inter)
    assert (q_out[cu[-1]:] == 7.0).all()
    assert (q_out[torch.from_numpy((seq >= 0) & (pos < 0)).cuda()] == 0).all()
    stored = np.zeros((cache.pages, page), bool)
    for name, x, w, heads in (("q", q, wq, hq), ("k", k, wk, kv)):
        w = None if w is None else w.cpu().numpy()
        ref = paged.norm_rotate(_np(x), w, *args)
        plain = paged.norm_rotate(_np(x), w, 1e-6, pos, None, inter)
        size = np.abs(plain).max(-1, keepdims=True) * 2
        tol = U[dt] * np.abs(ref) + 2e-6 * size
        if name == "q":
            have = _np(q_out)
        else:
            have = np.zeros_like(ref)
            for i in np.flatnonzero(live):
                p, r = cache.table[seq[i], pos[i] // page], pos[i] % page
                stored[p, r] = True
                have[i] = _np(cache.kd[p, :, r])
                assert torch.equal(cache.vd[p, :, r], v[i])
        assert (np.abs(have - ref)[live] <= tol[live]).all(), name
    keep = torch.from_numpy(~stored).cuda()[:, None, :, None].expand(cache.k.shape)
    for was, now in zip(before, (cache.kd, cache.vd)):
        assert torch.equal(was[keep].view(torch.int16), now[keep].view(torch.int16))


def test_append_far_positions_and_in_place(cuda):
    """Angles at a position near 10^6; q_out is q; one token per sequence."""
    from hybrid_llm_b200 import kernels
    page, far = 256, 999_937
    width = far // page + 1
    table = torch.zeros(2, width, dtype=torch.int32, device="cuda")
    table[0, far // page], table[1, 0] = 1, 0
    kp, vp = (torch.zeros(2, 2, page, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    lengths = torch.tensor([far + 1, 3], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(2, 4, 128, generator=g, device="cuda").half()
    k = torch.randn(2, 2, 128, generator=g, device="cuda").half()
    inv = (10000.0 ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64)).float()
    ref = paged.norm_rotate(_np(q), None, 0, [far, 2], inv.cpu().numpy(), False)
    tol = U[torch.float16] * np.abs(ref) + 4e-6 * np.abs(_np(q)).max()
    out = kernels.paged_append(q, k, k, kp, vp, table, lengths, inv_freq=inv, q_out=q)
    kernels.check_device_status()
    assert out is q and (np.abs(_np(q) - ref) <= tol).all()
    assert torch.equal(vp[1, :, far % page], k[0])


def test_append_bad_page_is_reported_and_skipped(cuda):
    from hybrid_llm_b200 import kernels
    kp = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    x = torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[0], [-1], [2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda")
    kernels.paged_append(x, x, x, kp, vp, table, lengths)
    with pytest.raises(RuntimeError, match="invalid argument"):
        kernels.check_device_status()
    kernels.check_device_status()  # reported once
    assert float(vp.sum()) == 64.0


# ------------------------------------------------------------------- decode
DECODE = [
    # lengths, hq, kv, dim, page, softcap, window, alibi, layout
    ([1], 1, 1, 128, 16, 0, 0, False, "hnd"),
    ([0], 4, 2, 64, 16, 0, 0, False, "hnd"),
    ([0, 1, 0, 15, 16, 17, 0], 4, 2, 128, 16, 0, 0, False, "hnd"),
    ([31, 32, 33, 1000], 6, 2, 64, 16, 0, 0, False, "nhd"),
    ([777], 8, 1, 128, 64, 30.0, 0, False, "hnd"),
    ([513, 64, 63, 65], 5, 5, 64, 32, 0, 0, True, "hnd"),
    ([300, 5, 999], 7, 1, 128, 128, 20.0, 100, True, "nhd"),
    ([256, 257, 1], 20, 1, 64, 256, 0, 1, False, "hnd"),
    ([400] * 40, 16, 8, 64, 16, 0, 37, False, "hnd"),
    ([5000, 3], 33, 1, 128, 16, 0, 0, False, "hnd"),
    (list(range(0, 330, 3)), 4, 4, 128, 32, 50.0, 0, False, "hnd"),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lengths,hq,kv,dim,page,softcap,window,alibi,layout", DECODE)
def test_decode(cuda, dtype, lengths, hq, kv, dim, page, softcap, window, alibi, layout):
    from hybrid_llm_b200 import kernels
    dt = DT[dtype]
    cache = Cache(lengths, kv, dim, page, dt, seed=len(lengths) + hq, layout=layout)
    g = torch.Generator().manual_seed(2)
    b = len(lengths)
    wide = torch.randn(b, hq + 1, dim + 8, generator=g).to(dt).cuda()
    q = wide[:, 1:, 8:]  # strided rows and heads
    slopes = torch.rand(hq, generator=g).cuda() if alibi else None
    out = torch.full((b, hq, dim), 9.0, dtype=dt, device="cuda")
    lse = torch.full((b, hq), 9.0, device="cuda")
    kernels.paged_decode(q, cache.kd, cache.vd, cache.td, cache.ld, softcap=softcap,
                         window=window, slopes=slopes, out=out, lse=lse)
    kernels.check_device_status()
    _check(out, lse, cache, q, np.arange(b + 1), dt, softcap=softcap, window=window,
           slopes=None if slopes is None else _np(slopes))


def test_decode_window_pages_may_be_gone(cuda):
    """Pages wholly before the window are not looked at: their entries may be anything."""
    from hybrid_llm_b200 import kernels
    cache = Cache([500, 90], 2, 64, 16, torch.bfloat16, seed=3)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    table = cache.td.clone()
    table[0, :(500 - 50) // 16] = -7
    table[1, :(90 - 50) // 16] = 1 << 30
    out = kernels.paged_decode(q, cache.kd, cache.vd, table, cache.ld, window=50)
    kernels.check_device_status()
    _check(out, None, cache, q, np.arange(3), torch.bfloat16, window=50)


def test_bad_pages_and_lengths_are_reported(cuda):
    """A page number out of range, and a length that the table cannot hold, reach no memory."""
    from hybrid_llm_b200 import kernels
    cache = Cache([40, 20], 1, 64, 16, torch.bfloat16, seed=4, pad=0)
    q = torch.randn(2, 1, 64, device="cuda").bfloat16()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for entry in (cache.pages, -1, 1 << 30):
        table = cache.td.clone()
        table[0, 1] = entry
        for call in (lambda: kernels.paged_decode(q, cache.kd, cache.vd, table, cache.ld),
                     lambda: kernels.paged_prefill(q, cache.kd, cache.vd, table, cache.ld, cu)):
            call()
            with pytest.raises(RuntimeError, match="invalid argument"):
                kernels.check_device_status()


def test_decode_long_context_many_splits(cuda):
    """One sequence over every worker, scores far apart (the maximum moves late)."""
    from hybrid_llm_b200 import kernels
    cache = Cache([20011], 2, 128, 64, torch.bfloat16, seed=6)
    g = torch.Generator().manual_seed(8)
    q = (torch.randn(1, 6, 128, generator=g) * 6).bfloat16().cuda()
    lse = torch.empty(1, 6, device="cuda")
    out = kernels.paged_decode(q, cache.kd, cache.vd, cache.td, cache.ld, lse=lse)
    kernels.check_device_status()
    ref, mag, _ = paged.attention(_np(q), cache.k_ref, cache.v_ref, cache.table, cache.lengths,
                                  [0, 1], scale=128 ** -0.5)
    # six times the scores: 6 2^-13 of their rounding
    tol = U[torch.bfloat16] * np.abs(ref) + (U[torch.bfloat16] + 6 * 2.0 ** -12) * mag
    assert (np.abs(_np(out) - ref) <= tol).all()
    again = kernels.paged_decode(q, cache.kd, cache.vd, cache.td, cache.ld)
    assert torch.equal(out, again)


# ------------------------------------------------------------------ prefill
PREFILL = [
    # new, context, hq, kv, dim, page, softcap, window, alibi, prefix, layout
    ([1], [0], 1, 1, 128, 16, 0, 0, False, None, "hnd"),
    ([7], [0], 4, 2, 64, 16, 0, 0, False, None, "hnd"),
    ([130, 1, 0, 257], [0, 300, 50, 3], 4, 4, 128, 32, 0, 0, False, None, "hnd"),
    ([128, 256, 64], [0, 0, 64], 2, 1, 64, 64, 0, 0, False, None, "nhd"),
    ([600], [0], 3, 1, 128, 128, 30.0, 0, False, None, "hnd"),
    ([90, 333], [1000, 17], 5, 1, 64, 16, 0, 0, True, None, "hnd"),
    ([300, 40], [200, 700], 8, 2, 128, 16, 20.0, 100, True, None, "nhd"),
    ([257, 100], [0, 500], 4, 4, 64, 256, 0, 1, False, None, "hnd"),
    ([200, 300, 50], [0, 100, 400], 4, 1, 128, 64, 0, 0, False, [150, 0, 9999], "hnd"),
    ([150, 65], [20, 0], 6, 3, 64, 32, 10.0, 0, True, [165, 64], "nhd"),
    ([5, 3], [2000, 3000], 16, 1, 128, 16, 0, 0, False, None, "hnd"),
    ([33], [100], 33, 1, 64, 16, 0, 50, False, None, "hnd"),
    ([3], [40], 128, 1, 64, 16, 0, 0, False, None, "hnd"),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("new,context,hq,kv,dim,page,softcap,window,alibi,prefix,layout", PREFILL)
def test_prefill(cuda, dtype, new, context, hq, kv, dim, page, softcap, window, alibi, prefix,
                 layout):
    from hybrid_llm_b200 import kernels
    dt = DT[dtype]
    lengths = [a + b for a, b in zip(new, context)]
    cache = Cache(lengths, kv, dim, page, dt, seed=sum(new) + hq, layout=layout)
    g = torch.Generator().manual_seed(3)
    cu = np.concatenate([[0], np.cumsum(new)])
    n = cu[-1] + 3  # rows behind the last sequence
    wide = torch.randn(n, hq + 1, dim + 8, generator=g).to(dt)
    wide[cu[-1]:] = float("nan")
    q = wide.cuda()[:, 1:, 8:]
    slopes = torch.rand(hq, generator=g).cuda() if alibi else None
    pre = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    out = torch.full((n, hq, dim), 9.0, dtype=dt, device="cuda")
    lse = torch.full((n, hq), 9.0, device="cuda")
    kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld,
                          torch.from_numpy(cu.astype(np.int32)).cuda(), softcap=softcap,
                          window=window, slopes=slopes, prefix=pre, out=out, lse=lse)
    kernels.check_device_status()
    assert (out[cu[-1]:] == 9.0).all() and (lse[cu[-1]:] == 9.0).all()
    _check(out, lse, cache, q[:cu[-1]], cu, dt, softcap=softcap, window=window,
           slopes=None if slopes is None else _np(slopes), prefix=prefix)


def test_prefill_rows_without_keys(cuda):
    """Tokens before position 0 (a length shorter than the tokens) see nothing: zeros."""
    from hybrid_llm_b200 import kernels
    cache = Cache([4, 0, 130], 1, 64, 16, torch.bfloat16, seed=9)
    new = [10, 5, 140]
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.randn(cu[-1], 2, 64, device="cuda").bfloat16()
    pre = torch.tensor([3, 2, 100], dtype=torch.int32, device="cuda")
    lse = torch.empty(cu[-1], 2, device="cuda")
    for p in (None, pre):
        out = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld,
                                    torch.from_numpy(cu.astype(np.int32)).cuda(), prefix=p, lse=lse)
        kernels.check_device_status()
        _check(out, lse, cache, q, cu, torch.bfloat16, prefix=None if p is None else [3, 2, 100])
        assert (out[:6] == 0).all() and (lse[:6] == -float("inf")).all()


def test_prefill_many_units_and_moving_maximum(cuda):
    """More units than SMs, ragged, with a few large scores; repeated bit for bit."""
    from hybrid_llm_b200 import kernels
    new = [900, 1, 513, 256, 700, 31, 640, 333]
    context = [0, 250, 128, 77, 0, 0, 1, 500]
    lengths = [a + b for a, b in zip(new, context)]
    cache = Cache(lengths, 8, 64, 32, torch.bfloat16, seed=12)
    cu = np.concatenate([[0], np.cumsum(new)])
    g = torch.Generator().manual_seed(4)
    q = torch.randn(cu[-1], 16, 64, generator=g)
    q[::97] *= 6
    q = q.bfloat16().cuda()
    cud = torch.from_numpy(cu.astype(np.int32)).cuda()
    out = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, cud)
    kernels.check_device_status()
    ref, mag, _ = paged.attention(_np(q), cache.k_ref, cache.v_ref, cache.table, lengths, cu,
                                  scale=0.125)
    tol = U[torch.bfloat16] * np.abs(ref) + (U[torch.bfloat16] + 6 * 2.0 ** -12) * mag
    assert (np.abs(_np(out) - ref) <= tol).all()
    for _ in range(4):
        assert torch.equal(out, kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, cud))


def test_prefill_one_token_equals_decode(cuda):
    """One new token per sequence through both operators, within both roundings."""
    from hybrid_llm_b200 import kernels
    cache = Cache([77, 1, 300], 2, 128, 16, torch.bfloat16, seed=13)
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    a = kernels.paged_decode(q, cache.kd, cache.vd, cache.td, cache.ld)
    b = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, cu)
    kernels.check_device_status()
    for x in (a, b):
        _check(x, None, cache, q, np.arange(4), torch.bfloat16)


# ----------------------------------------------------------------- together
def test_conversation(cuda):
    """A prompt in two chunks, then tokens one by one: append, attend, per step."""
    from hybrid_llm_b200 import kernels
    rng = np.random.default_rng(20)
    hq, kv, dim, page, b = 4, 2, 64, 16, 3
    chunks = [[40, 7, 100], [21, 30, 0]] + [[1, 1, 1]] * 5
    total = np.sum(chunks, 0)
    cache = Cache(list(total), kv, dim, page, torch.bfloat16, seed=21)
    inv = torch.tensor(10000.0 ** (-np.arange(32) / 32), dtype=torch.float32).cuda()
    wq, wk = (torch.from_numpy(rng.normal(1, 0.2, dim).astype(np.float32)).cuda() for _ in range(2))
    done = np.zeros(b, np.int64)
    k_ref, v_ref = np.zeros_like(cache.k_ref), np.zeros_like(cache.v_ref)
    for new in chunks:
        done = done + new
        cu = np.concatenate([[0], np.cumsum(new)])
        n = cu[-1]
        ld = torch.from_numpy(done.astype(np.int32)).cuda()
        cud = torch.from_numpy(cu.astype(np.int32)).cuda()
        x = torch.from_numpy(rng.normal(size=(n, hq + 2 * kv, dim)).astype(np.float32)).bfloat16().cuda()
        q, k, v = x[:, :hq], x[:, hq:hq + kv], x[:, hq + kv:]
        single = max(new) == 1
        qr = kernels.paged_append(q, k, v, cache.kd, cache.vd, cache.td, ld,
                                  cu_q=None if single else cud, inv_freq=inv, q_norm=wq, k_norm=wk)
        out = (kernels.paged_decode(qr, cache.kd, cache.vd, cache.td, ld) if single else
               kernels.paged_prefill(qr, cache.kd, cache.vd, cache.td, ld, cud))
        kernels.check_device_status()
        # the oracle attends over the rows that the append stored
        seq, pos = paged.positions(cu, done, n)
        kk = paged.norm_rotate(_np(k), wk.cpu().numpy(), 1e-6, pos, inv.cpu().numpy(), False)
        for i in range(n):
            p, r = cache.table[seq[i], pos[i] // page], pos[i] % page
            have = _np(cache.kd[p, :, r])
            assert np.abs(have - kk[i]).max() <= 2.0 ** -8 * np.abs(kk[i]).max() + 1e-5
            k_ref[p, :, r], v_ref[p, :, r] = have, _np(v[i])
        cache.k_ref, cache.v_ref, cache.lengths = k_ref, v_ref, done
        _check(out, None, cache, qr, cu, torch.bfloat16)


def test_captured_step_follows_its_inputs(cuda):
    """A captured append + decode step replayed with growing lengths, on another
    stream than its inputs', with a second graph of the same kind between."""
    from hybrid_llm_b200 import kernels
    page, dim, hq, kv = 16, 128, 4, 2
    lengths = [200, 31]
    caches = [Cache(lengths, kv, dim, page, torch.bfloat16, seed=s) for s in (30, 31)]
    stream = torch.cuda.Stream()
    graphs = []
    for c in caches:
        c.x = torch.zeros(2, hq + 2 * kv, dim, dtype=torch.bfloat16, device="cuda")
        c.n = torch.tensor([1, 1], dtype=torch.int32, device="cuda")

        def step(c=c):
            q = kernels.paged_append(c.x[:, :hq], c.x[:, hq:hq + kv], c.x[:, hq + kv:], c.kd, c.vd,
                                     c.td, c.n)
            return kernels.paged_decode(q, c.kd, c.vd, c.td, c.n)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                c.out = step()
        graphs.append(g)
        first = c.table[:, 0]  # the uncaptured step stored zero rows at position 0
        c.k_ref[first, :, 0], c.v_ref[first, :, 0] = 0.0, 0.0
    g = torch.Generator().manual_seed(5)
    for length in ([150, 9], [151, 10], [200, 31]):
        for c, graph in zip(caches, graphs):
            c.x.copy_(torch.randn(c.x.shape, generator=g).bfloat16())
            c.n.copy_(torch.tensor(length, dtype=torch.int32))
            graph.replay()
        torch.cuda.synchronize()
        kernels.check_device_status()
        for c in caches:
            for b in range(2):
                p, r = c.table[b, (length[b] - 1) // page], (length[b] - 1) % page
                c.k_ref[p, :, r], c.v_ref[p, :, r] = _np(c.x[b, hq:hq + kv]), _np(c.x[b, hq + kv:])
            c.lengths = np.asarray(length)
            _check(c.out, None, c, c.x[:, :hq], np.arange(3), torch.bfloat16)


def test_two_streams_at_once(cuda):
    """Two decodes and two prefills in flight on two streams, each with its own scratch."""
    from hybrid_llm_b200 import kernels
    cache = Cache([3000, 40], 2, 64, 16, torch.bfloat16, seed=40)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    cu = torch.arange(3, dtype=torch.int32, device="cuda")
    want = kernels.paged_decode(q, cache.kd, cache.vd, cache.td, cache.ld)
    want_p = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, cu)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((kernels.paged_decode(q, cache.kd, cache.vd, cache.td, cache.ld),
                            kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, cu)))
    torch.cuda.synchronize()
    kernels.check_device_status()
    for d, p in got:
        assert torch.equal(d, want) and torch.equal(p, want_p)


def test_refusals(cuda):
    from hybrid_llm_b200 import kernels
    cache = Cache([40], 2, 64, 16, torch.bfloat16, seed=50)
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    ok = (cache.kd, cache.vd, cache.td, cache.ld)
    kv = q[:, :2]

    def refused(f, *a, **kw):
        with pytest.raises(ValueError):
            f(*a, **kw)
    for f, tail in ((kernels.paged_decode, ()), (kernels.paged_prefill, (cu,))):
        refused(f, q.half(), *ok, *tail)
        refused(f, q[:, :3], *ok, *tail)                       # 3 heads over 2
        refused(f, q[..., :32], *ok, *tail)
        refused(f, q, cache.kd[..., :32], cache.vd[..., :32], cache.td, cache.ld, *tail)
        refused(f, q, cache.kd, cache.vd.transpose(1, 2).contiguous().transpose(1, 2), cache.td,
                cache.ld, *tail)
        refused(f, q, cache.kd[:, :, :8], cache.vd[:, :, :8], cache.td, cache.ld, *tail)
        refused(f, q, cache.kd, cache.vd, cache.td.long(), cache.ld, *tail)
        refused(f, q, cache.kd, cache.vd, cache.td, cache.ld.long(), *tail)
        refused(f, q, *ok, *tail, scale=0.0)
        refused(f, q, *ok, *tail, scale=float("nan"))
        refused(f, q, *ok, *tail, softcap=-1.0)
        refused(f, q, *ok, *tail, window=-1)
        refused(f, q, *ok, *tail, slopes=torch.ones(3, device="cuda"))
        refused(f, q, *ok, *tail, out=torch.empty(1, 4, 64, device="cuda"))
        refused(f, q, *ok, *tail, lse=torch.empty(4, device="cuda"))
        with pytest.raises(RuntimeError):
            f(q.cpu(), *ok, *tail)
    refused(kernels.paged_decode, torch.cat([q, q]), *ok)
    refused(kernels.paged_prefill, q, *ok, cu.long())
    refused(kernels.paged_prefill, q, *ok, cu, window=4, prefix=cache.ld)
    refused(kernels.paged_append, q, kv, kv[:, :1], *ok)
    refused(kernels.paged_append, torch.cat([q, q]), torch.cat([kv, kv]), torch.cat([kv, kv]), *ok)
    refused(kernels.paged_append, q, kv, kv, *ok, inv_freq=torch.ones(12, device="cuda"))
    refused(kernels.paged_append, q, kv, kv, *ok, inv_freq=torch.ones(40, device="cuda"))
    refused(kernels.paged_append, q, kv, kv, *ok, q_norm=torch.ones(32, device="cuda"))


def test_empty_calls(cuda):
    """No sequences, or sequences without tokens."""
    from hybrid_llm_b200 import kernels
    cache = Cache([40], 2, 64, 16, torch.bfloat16, seed=50)
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    t, l = cache.td[:0], cache.ld[:0]
    assert kernels.paged_decode(q, cache.kd, cache.vd, t, l).shape == q.shape
    assert kernels.paged_prefill(q, cache.kd, cache.vd, t, l, none).shape == q.shape
    assert kernels.paged_append(q, q[:, :2], q[:, :2], cache.kd, cache.vd, t, l,
                                cu_q=none).shape == q.shape
    two = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, two).shape == q.shape
    row = torch.full((1, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    out = row.clone()
    kernels.paged_prefill(row, cache.kd, cache.vd, cache.td, cache.ld, two, out=out)
    assert torch.equal(out, row)
    kernels.check_device_status()


def test_cache_object_serves_a_batch(cuda):
    """PagedKVCache: prompts, steps, a row that ends and another that takes its pages."""
    from hybrid_llm_b200.state import PagedKVCache
    hq, kv, dim = 4, 2, 64
    c = PagedKVCache(kv, dim, batch=2, pages=12, page_size=16, layers=2)
    g = torch.Generator().manual_seed(6)
    rows = {0: [], 1: []}  # (key, value) of every position

    def check(new, cu_q):
        n = sum(new)
        x = torch.randn(n, hq + 2 * kv, dim, generator=g).bfloat16().cuda()
        for layer in range(2):
            q = c.append(layer, x[:, :hq], x[:, hq:hq + kv], x[:, hq + kv:], cu_q)
            out = c.attend(layer, q, cu_q)
            if layer == 0:
                at = 0
                for b, t in enumerate(new):
                    rows[b] += [(x[i, hq:hq + kv], x[i, hq + kv:]) for i in range(at, at + t)]
                    at += t
            at = 0
            for b, t in enumerate(new):
                if t == 0:
                    continue
                k, v = (_np(torch.stack([r[j] for r in rows[b]])) for j in (0, 1))
                ref, mag, _ = paged.attention(
                    _np(q[at:at + t]), k.transpose(1, 0, 2)[None], v.transpose(1, 0, 2)[None],
                    np.zeros((1, 1), int), [len(rows[b])], [0, t], scale=dim ** -0.5)
                _close(out[at:at + t], ref, mag, torch.bfloat16, [1], 1)
                at += t

    check([50, 20], c.extend([50, 20]))
    for _ in range(3):
        c.extend([1, 1])
        check([1, 1], None)
    check([0, 30], c.extend([0, 30]))
    c.release([0])
    rows[0] = []
    check([90, 1], c.extend([90, 1]))
    assert c.free_pages == 12 - 6 - 4
    from hybrid_llm_b200 import kernels
    kernels.check_device_status()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16)])
def test_decode_one_cta_per_head(cuda, dtype, dim, page):
    """Enough rows that every sequence and kv head has a CTA of its own."""
    from hybrid_llm_b200 import kernels
    rng = np.random.default_rng(dim)
    lengths = [0, 1, 800] + [int(x) for x in rng.integers(0, 700, 160)]
    cache = Cache(lengths, 4, dim, page, DT[dtype], seed=60, pad=0)
    q = torch.randn(len(lengths), 12, dim, device="cuda").to(DT[dtype])
    lse = torch.empty(len(lengths), 12, device="cuda")
    out = kernels.paged_decode(q, cache.kd, cache.vd, cache.td, cache.ld, lse=lse, window=300)
    kernels.check_device_status()
    _check(out, lse, cache, q, np.arange(len(lengths) + 1), DT[dtype], window=300)


def test_tables_with_a_row_stride(cuda):
    """block_table a slice of a wider table, through all three calls."""
    from hybrid_llm_b200 import kernels
    cache = Cache([70, 9], 2, 64, 16, torch.bfloat16, seed=61, pad=0)
    wide = torch.full((2, cache.table.shape[1] + 5), -9, dtype=torch.int32, device="cuda")
    table = wide[:, 3:3 + cache.table.shape[1]]
    table.copy_(cache.td)
    x = torch.randn(2, 8, 64, device="cuda").bfloat16()
    q = kernels.paged_append(x[:, :4], x[:, 4:6], x[:, 6:], cache.kd, cache.vd, table, cache.ld)
    for b, n in enumerate((70, 9)):
        p, r = cache.table[b, (n - 1) // 16], (n - 1) % 16
        cache.k_ref[p, :, r], cache.v_ref[p, :, r] = _np(x[b, 4:6]), _np(x[b, 6:])
    cu = torch.arange(3, dtype=torch.int32, device="cuda")
    for out in (kernels.paged_decode(q, cache.kd, cache.vd, table, cache.ld),
                kernels.paged_prefill(q, cache.kd, cache.vd, table, cache.ld, cu)):
        _check(out, None, cache, q, np.arange(3), torch.bfloat16)
    kernels.check_device_status()


@pytest.mark.parametrize("width", [2, 40])
def test_prefill_of_very_many_sequences(cuda, width):
    """20,000 sequences of one token (several chunk sums share one): as decode."""
    from hybrid_llm_b200 import kernels
    g = torch.Generator(device="cuda").manual_seed(7)
    b, pages = 20000, 64
    kp, vp = (torch.randn(pages, 1, 16, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(b, 1, 64, generator=g, device="cuda").bfloat16()
    table = torch.randint(0, pages, (b, width), generator=g, device="cuda", dtype=torch.int32)
    lengths = torch.randint(0, 33, (b,), generator=g, device="cuda", dtype=torch.int32)
    cu = torch.arange(b + 1, dtype=torch.int32, device="cuda")
    a = kernels.paged_prefill(q, kp, vp, table, lengths, cu)
    d = kernels.paged_decode(q, kp, vp, table, lengths)
    kernels.check_device_status()
    # both round their weights and outputs: twice 2^-8 of each, values up to 6
    assert (a.float() - d.float()).abs().max() <= 4 * 2.0 ** -8 * 6
    # the mean over 1.2 million values is unbiased, so a lost sequence shows
    assert (a.float() - d.float()).abs().mean() < 2.0 ** -8
    assert (a[lengths == 0] == 0).all()


def test_prefill_many_groups_of_sequences(cuda):
    """75 sequences in three groups, pieces in several chunks, some empty."""
    from hybrid_llm_b200 import kernels
    rng = np.random.default_rng(8)
    new = [int(x) for x in rng.integers(0, 60, 75)]
    new[3], new[40], new[74] = 700, 0, 333
    context = [int(x) for x in rng.integers(0, 900, 75)]
    lengths = [a + c for a, c in zip(new, context)]
    cache = Cache(lengths, 2, 64, 32, torch.bfloat16, seed=62)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.randn(cu[-1], 14, 64, device="cuda").bfloat16()
    lse = torch.empty(cu[-1], 14, device="cuda")
    out = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld,
                                torch.from_numpy(cu.astype(np.int32)).cuda(), lse=lse, softcap=8.0)
    kernels.check_device_status()
    _check(out, lse, cache, q, cu, torch.bfloat16, softcap=8.0)


def test_non_finite_values_reach_only_their_readers(cuda):
    """A NaN or an infinity in a query or a key spoils that row (or the rows that
    see the key), in decode and prefill; nothing else."""
    from hybrid_llm_b200 import kernels
    cache = Cache([200, 300], 1, 64, 16, torch.bfloat16, seed=63)
    new = [40, 300]
    cu = np.concatenate([[0], np.cumsum(new)])
    cud = torch.from_numpy(cu.astype(np.int32)).cuda()
    q = torch.randn(cu[-1], 2, 64, device="cuda").bfloat16()
    clean = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, cud)
    bad = q.clone()
    bad[17, 1, 5] = float("nan")
    out = kernels.paged_prefill(bad, cache.kd, cache.vd, cache.td, cache.ld, cud)
    assert out[17, 1].isnan().all()
    keep = torch.ones(cu[-1], 2, dtype=torch.bool, device="cuda")
    keep[17, 1] = False
    assert torch.equal(out[keep], clean[keep])
    kd = cache.kd.clone()
    kd[cache.table[1, 250 // 16], 0, 250 % 16, 3] = float("nan")
    for softcap in (0.0, 20.0):
        clean = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, cud, softcap=softcap)
        out = kernels.paged_prefill(q, kd, cache.vd, cache.td, cache.ld, cud, softcap=softcap)
        assert torch.equal(out[:40 + 250], clean[:40 + 250]) and out[40 + 250:].isnan().all()
        one = kernels.paged_decode(q[:2], kd, cache.vd, cache.td, cache.ld, softcap=softcap)
        assert not one[0].isnan().any() and one[1].isnan().all()
    kernels.check_device_status()


def test_largest_window_and_lengths_beyond_the_table(cuda):
    """A window of 2^31 - 1 is none; attention counts what the table holds, append
    reports a token that has no page."""
    from hybrid_llm_b200 import kernels
    cache = Cache([64, 700], 2, 128, 16, torch.bfloat16, seed=64, pad=0)
    # the shorter row's table is filled up so that every position has a page
    cache.table[0] = np.where(cache.table[0] < 0, cache.table[1], cache.table[0])
    td = torch.from_numpy(cache.table).cuda()
    held = cache.table.shape[1] * 16
    cu = torch.tensor([0, 3, 40], dtype=torch.int32, device="cuda")
    q = torch.randn(40, 4, 128, device="cuda").bfloat16()
    w = 2 ** 31 - 1
    assert torch.equal(kernels.paged_prefill(q, cache.kd, cache.vd, td, cache.ld, cu, window=w),
                       kernels.paged_prefill(q, cache.kd, cache.vd, td, cache.ld, cu))
    assert torch.equal(kernels.paged_decode(q[:2], cache.kd, cache.vd, td, cache.ld, window=w),
                       kernels.paged_decode(q[:2], cache.kd, cache.vd, td, cache.ld))
    kernels.check_device_status()
    kd, vd = cache.kd.nan_to_num(0, 0, 0), cache.vd.nan_to_num(0, 0, 0)
    full = torch.tensor([held, held], dtype=torch.int32, device="cuda")
    beyond = torch.tensor([held + 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    assert torch.equal(kernels.paged_decode(q[:2], kd, vd, td, beyond),
                       kernels.paged_decode(q[:2], kd, vd, td, full))
    assert torch.equal(kernels.paged_prefill(q, kd, vd, td, beyond, cu),
                       kernels.paged_prefill(q, kd, vd, td, full, cu))
    kernels.check_device_status()
    before = kd.clone()
    kernels.paged_append(q[:2], q[:2, :2], q[:2, :2], kd, vd, td, beyond)
    with pytest.raises(RuntimeError, match="invalid argument"):
        kernels.check_device_status()
    assert torch.equal(kd, before)


def test_captured_step_of_the_cache_object(cuda):
    """Prompts, a captured append + attend that counts the lengths up, advance, a
    row released, another one extended, and the same graph again."""
    from hybrid_llm_b200 import kernels
    from hybrid_llm_b200.state import PagedKVCache
    hq, kv, dim, b = 4, 2, 64, 3
    c = PagedKVCache(kv, dim, batch=b, pages=24, page_size=16)
    kernels.device_status(c.device)
    g = torch.Generator().manual_seed(9)
    rows = [[] for _ in range(b)]  # (key, value) of every position

    def tokens(n):
        return torch.randn(n, hq + 2 * kv, dim, generator=g).bfloat16().cuda()

    def split(x):
        return x[:, :hq], x[:, hq:hq + kv], x[:, hq + kv:]

    def check(out, x, new):
        at = 0
        for r, t in enumerate(new):
            rows[r] += [(x[i, hq:hq + kv], x[i, hq + kv:]) for i in range(at, at + t)]
            if t:
                k, v = (_np(torch.stack([p[j] for p in rows[r]])) for j in (0, 1))
                ref, mag, _ = paged.attention(
                    _np(x[at:at + t, :hq]), k.transpose(1, 0, 2)[None], v.transpose(1, 0, 2)[None],
                    np.zeros((1, 1), int), [len(rows[r])], [0, t], scale=dim ** -0.5)
                _close(out[at:at + t], ref, mag, torch.bfloat16, [1], 1)
            at += t

    def prompt(new):
        cu, x = c.extend(new), tokens(sum(new))
        q, k, v = split(x)
        check(c.attend(0, c.append(0, q, k, v, cu), cu), x, new)

    prompt([20, 5, 40])
    x = tokens(b)
    live = torch.zeros(b, dtype=torch.int32, device="cuda")
    c.extend([1, 1, 1])
    q, k, v = split(x)
    check(c.attend(0, c.append(0, q, k, v)), x.clone(), [1, 1, 1])

    def step():
        c.lengths.add_(live)
        q, k, v = split(x)
        return c.attend(0, c.append(0, q, k, v))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()

    def replay(times, new):
        c.reserve([times * n for n in new])
        live.copy_(torch.tensor(new, dtype=torch.int32))
        for _ in range(times):
            x.copy_(tokens(b))
            graph.replay()
            for r, n in enumerate(new):
                if n == 0:
                    assert (out[r] == 0).all()
            keep = [r for r in range(b) if new[r]]
            check(out[keep], x[keep], new)
        c.advance([times * n for n in new])

    replay(12, [1, 1, 1])
    assert c.lengths.tolist() == [33, 18, 53]
    prompt([0, 7, 0])
    c.release([0])
    rows[0] = []
    replay(20, [0, 1, 1])
    prompt([33, 1, 2])
    replay(3, [1, 1, 1])
    assert c.lengths.tolist() == [36, 49, 78]
    kernels.check_device_status()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 70, 100])
def test_prefill_window_where_tokens_have_no_position(cuda, window):
    """A piece that begins before position 0, under the largest windows: its later
    tokens see their keys."""
    from hybrid_llm_b200 import kernels
    cache = Cache([4, 0, 130], 1, 64, 16, torch.bfloat16, seed=65)
    new = [10, 5, 140]
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.randn(cu[-1], 2, 64, device="cuda").bfloat16()
    lse = torch.empty(cu[-1], 2, device="cuda")
    out = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld,
                                torch.from_numpy(cu.astype(np.int32)).cuda(), window=window, lse=lse)
    kernels.check_device_status()
    _check(out, lse, cache, q, cu, torch.bfloat16, window=window)
    assert (out[:6] == 0).all() and (out[6:10] != 0).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("softcap,size", [(0.5, 8.0), (3.0, 12.0), (1000.0, 2.0), (1e5, 8.0)])
@pytest.mark.parametrize("dim,page,width", [(64, 16, 0), (128, 64, 900)])
def test_caps_far_from_the_scores(cuda, dtype, softcap, size, dim, page, width):
    """Scores past the cap (saturated beside unsaturated ones in a warp) and caps far
    above them, by both operators; whole and cut units.  `size` times the scores of
    the file's tolerance, so `size` times its score terms; tanh is off by 2^-19 of
    itself at most, below that."""
    from hybrid_llm_b200 import kernels
    dt = DT[dtype]
    new, context = [150, 3, 40], [0, 200 + width, 90]
    lengths = [a + b for a, b in zip(new, context)]
    cache = Cache(lengths, 2, dim, page, dt, seed=66 + dim)
    cu = np.concatenate([[0], np.cumsum(new)])
    g = torch.Generator().manual_seed(10)
    q = torch.randn(cu[-1], 6, dim, generator=g)
    q[::3] *= size  # a third of the rows
    q = q.to(dt).cuda()
    last = [int(x) - 1 for x in cu[1:]]
    u, score = U[dt], size * 2.0 ** -13
    for call, rows, begin in (
            (lambda q, **o: kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld,
                                                  torch.from_numpy(cu.astype(np.int32)).cuda(), **o),
             list(range(cu[-1])), cu),
            (lambda q, **o: kernels.paged_decode(q, cache.kd, cache.vd, cache.td, cache.ld, **o),
             last, np.arange(4))):
        qr = q[rows].contiguous()
        lse = torch.empty(len(rows), 6, device="cuda")
        out = call(qr, softcap=softcap, lse=lse)
        kernels.check_device_status()
        ref, mag, l_ref = paged.attention(_np(qr), cache.k_ref, cache.v_ref, cache.table, lengths,
                                          begin, scale=dim ** -0.5, softcap=softcap)
        tol = u * np.abs(ref) + (u + 2 * score) * mag
        if dt is torch.float16:
            tol = tol + max(lengths) * 2.0 ** -25 * np.abs(cache.v_ref).max()
        assert (np.abs(_np(out) - ref) <= tol).all()
        assert (np.abs(_np(lse) - l_ref) <= score + 2.0 ** -20 * np.abs(l_ref)).all()


@pytest.mark.parametrize("packed", [False, True])
def test_append_idle_slots_are_zero(cuda, packed):
    """A token without a position: its query is zero with eps = 0, with a weight that
    is not finite and with query rows that are not; nothing is stored for it."""
    from hybrid_llm_b200 import kernels
    cache = Cache([0, 5, 0], 1, 64, 16, torch.bfloat16, seed=67)
    x = torch.randn(3, 4, 64, device="cuda").bfloat16()
    x[0, 0], x[2, 1, 3] = 0, float("nan")
    w = torch.ones(64, device="cuda")
    w[7] = float("inf")
    before = cache.kd.clone(), cache.vd.clone()
    cu = torch.arange(4, dtype=torch.int32, device="cuda") if packed else None
    inv = torch.tensor([float("inf")] * 8 + [1.0] * 8, device="cuda")
    q = kernels.paged_append(x[:, :2], x[:, 2:3], x[:, 3:], cache.kd, cache.vd, cache.td, cache.ld,
                             cu_q=cu, eps=0.0, q_norm=w, inv_freq=inv)
    kernels.check_device_status()
    assert (q[0] == 0).all() and (q[2] == 0).all() and not q[1].isfinite().all()
    p = int(cache.table[1, 0])
    assert torch.equal(cache.vd[p, :, 4], x[1, 3:])
    for was, now in zip(before, (cache.kd, cache.vd)):
        was[p, :, 4] = now[p, :, 4]
        assert torch.equal(was.view(torch.int16), now.view(torch.int16))


def test_packing_that_begins_behind_row_0(cuda):
    """cu_q of some sequences of a larger packed batch: the rows before cu_q[0] belong
    to none of them, in append as in prefill."""
    from hybrid_llm_b200 import kernels
    cache = Cache([40, 20], 2, 64, 16, torch.bfloat16, seed=68)
    cu = [7, 12, 15]
    cud = torch.tensor([0, 3, *cu, 18], dtype=torch.int32, device="cuda")[2:5]
    x = torch.randn(18, 8, 64, device="cuda").bfloat16()
    before = cache.kd.clone(), cache.vd.clone()
    q = torch.full((18, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    kernels.paged_append(x[:, :4], x[:, 4:6], x[:, 6:], cache.kd, cache.vd, cache.td, cache.ld,
                         cu_q=cud, q_out=q)
    kernels.check_device_status()
    assert (q[:7] == 7).all() and (q[15:] == 7).all() and torch.equal(q[7:15], x[7:15, :4])
    stored = torch.zeros(cache.pages, 16, dtype=torch.bool, device="cuda")
    for b in range(2):
        for i in range(cu[b], cu[b + 1]):
            at = int(cache.lengths[b]) - cu[b + 1] + i
            p, r = cache.table[b, at // 16], at % 16
            stored[int(p), r] = True
            assert torch.equal(cache.kd[p, :, r], x[i, 4:6]) and torch.equal(cache.vd[p, :, r], x[i, 6:])
            cache.k_ref[p, :, r], cache.v_ref[p, :, r] = _np(x[i, 4:6]), _np(x[i, 6:])
    keep = ~stored[:, None, :, None].expand(cache.k.shape)
    for was, now in zip(before, (cache.kd, cache.vd)):
        assert torch.equal(was[keep].view(torch.int16), now[keep].view(torch.int16))
    out = torch.full((18, 4, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, cud, out=out)
    kernels.check_device_status()
    assert (out[:7] == 9).all() and (out[15:] == 9).all()
    _check(out[7:], None, cache, q[7:15], np.asarray(cu) - 7, torch.bfloat16)


@pytest.mark.parametrize("far", [2 ** 25 + 128, 2 ** 30 - 4096])
def test_bias_and_window_at_far_positions(cuda, far):
    """Positions that fp32 does not hold: the same last keys as a short sequence's, seen
    through a window with a distance bias, behind a table of any other pages."""
    from hybrid_llm_b200 import kernels
    page, dim = 256, 64
    cache = Cache([700], 1, dim, page, torch.bfloat16, seed=69, pad=0)
    g = torch.Generator().manual_seed(11)
    q = torch.randn(9, 4, dim, generator=g).bfloat16().cuda()
    slopes = torch.tensor([0.9, 0.3, 0.05, -0.01], device="cuda")
    first = far // page  # pages before the short sequence's
    table = torch.full((1, first + cache.td.shape[1]), -1, dtype=torch.int32, device="cuda")
    table[:, first:] = cache.td
    lengths = cache.ld + first * page
    cu = np.asarray([0, 9])
    lse = torch.empty(9, 4, device="cuda")
    out = kernels.paged_prefill(q, cache.kd, cache.vd, table, lengths,
                                torch.tensor([0, 9], dtype=torch.int32, device="cuda"), window=300,
                                slopes=slopes, lse=lse)
    kernels.check_device_status()
    _check(out, lse, cache, q, cu, torch.bfloat16, window=300, slopes=_np(slopes))
    lse = torch.empty(1, 4, device="cuda")
    out = kernels.paged_decode(q[8:], cache.kd, cache.vd, table, lengths, window=300, slopes=slopes,
                               lse=lse)
    kernels.check_device_status()
    _check(out, lse, cache, q[8:], np.asarray([0, 1]), torch.bfloat16, window=300, slopes=_np(slopes))


def test_scores_that_fp32_does_not_hold_are_refused(cuda):
    """A cap that is 0 in fp32 is not taken for none; factors beyond fp32 are refused."""
    from hybrid_llm_b200 import kernels
    cache = Cache([40], 2, 64, 16, torch.bfloat16, seed=50)
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    ok = (cache.kd, cache.vd, cache.td, cache.ld)
    for f, tail in ((kernels.paged_decode, ()), (kernels.paged_prefill, (cu,))):
        for over in (dict(softcap=1e-50), dict(softcap=1e-39), dict(softcap=1e38),
                     dict(softcap=float("inf")), dict(softcap=1e39), dict(scale=1e-45),
                     dict(scale=3e38), dict(scale=4.0, softcap=1e-38), dict(scale=1e-30, softcap=1e9)):
            with pytest.raises(ValueError):
                f(q, *ok, *tail, **over)


def test_outputs_that_overlap_themselves_are_refused(cuda):
    """Expanded or overlapping outputs and pools have no place of their own for every
    element; any order of the dimensions, and gaps, are fine."""
    from hybrid_llm_b200 import kernels
    cache = Cache([40, 9], 2, 64, 16, torch.bfloat16, seed=50)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    kv = torch.randn(2, 2, 64, device="cuda").bfloat16()
    cu = torch.arange(3, dtype=torch.int32, device="cuda")
    at = (cache.td, cache.ld)
    pages = (cache.kd, cache.vd)
    flat = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    for strides in ((0, 64, 1), (256, 0, 1), (64, 64, 1), (256, 32, 1), (192, 64, 1), (8, 64, 1)):
        out = flat.as_strided((2, 4, 64), strides)
        for call in (lambda: kernels.paged_decode(q, *pages, *at, out=out),
                     lambda: kernels.paged_prefill(q, *pages, *at, cu, out=out),
                     lambda: kernels.paged_append(q, kv, kv, *pages, *at, q_out=out)):
            with pytest.raises(ValueError, match="overlaps itself"):
                call()
    pool = cache.kd[:, :1].expand(-1, 2, -1, -1)
    with pytest.raises(ValueError, match="overlaps itself"):
        kernels.paged_append(q, kv, kv, pool, pool, *at)
    want = kernels.paged_decode(q, *pages, *at)
    for strides in ((256, 64, 1), (64, 128, 1), (72, 144, 1), (1024, 128, 1)):
        out = flat.as_strided((2, 4, 64), strides)
        assert torch.equal(kernels.paged_decode(q, *pages, *at, out=out), want)
        assert torch.equal(out, want)
    one = flat.as_strided((1, 4, 64), (0, 64, 1))
    assert torch.equal(kernels.paged_decode(q[:1], *pages, cache.td[:1], cache.ld[:1], out=one), want[:1])
    kernels.check_device_status()


def test_fp16_keeps_many_small_weights(cuda):
    """40,000 keys 25.2 bits below the best one are 0.1 % of the weights' sum.  A weight
    is off by at most 2^-25 in units of 2^-kUp of the largest (subnormal), kUp = 12 in
    decode and 4 in prefill: n 2^-37 and n 2^-29 of max |v| beside the roundings."""
    from hybrid_llm_b200 import kernels
    n = 40000
    cache = Cache([n], 1, 64, 64, torch.float16, seed=70)
    g = torch.Generator().manual_seed(12)
    k, v = torch.zeros(n, 64), torch.rand(n, 64, generator=g) + 0.5
    k[0, 0], v[0] = 8.734375, 0.0            # scores 17.47 and 0
    for t, ref, x in ((cache.kd, cache.k_ref, k), (cache.vd, cache.v_ref, v)):
        x = x.half()
        for i, p in enumerate(cache.table[0, :n // 64]):
            t[int(p), 0] = x[64 * i:64 * i + 64].cuda()
            ref[int(p), 0] = _np(x[64 * i:64 * i + 64])
    q = torch.zeros(3, 2, 64)
    q[:, :, 0] = 16.0
    q = q.half().cuda()
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    u = U[torch.float16]
    for out, rows, up in ((kernels.paged_decode(q[2:], cache.kd, cache.vd, cache.td, cache.ld), [2], 12),
                          (kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld, cu),
                           [0, 1, 2], 4)):
        kernels.check_device_status()
        ref, mag, _ = paged.attention(_np(q[rows]), cache.k_ref, cache.v_ref, cache.table, [n],
                                      [0, len(rows)], scale=0.125)
        tol = u * np.abs(ref) + (u + 2 * 2.0 ** -12) * mag + n * 2.0 ** (-25 - up) * 1.5
        assert (np.abs(_np(out) - ref) <= tol).all() and (ref > 5e-4).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("pad", [0, 40])
@pytest.mark.parametrize("rise", [4.0, 12.0, 40.0])
def test_maximum_that_rises_late(cuda, dtype, pad, rise):
    """Keys are visited from the last to the first; the first ones score `rise` above the
    rest, beyond what the weights of the block may hold; whole and cut units.  Scores
    up to 10 + rise, so (1 + rise / 10) times the tolerance's score terms."""
    from hybrid_llm_b200 import kernels
    dt = DT[dtype]
    new, context = [70, 130, 1], [330, 200, 400]
    lengths = [a + b for a, b in zip(new, context)]
    cache = Cache(lengths, 1, 64, 16, dt, seed=71, pad=pad)
    for b in range(3):
        p = int(cache.table[b, 0])
        cache.kd[p, 0, :7, 0] = rise
        cache.k_ref[p, 0, :7, 0] = rise
    cu = np.concatenate([[0], np.cumsum(new)])
    g = torch.Generator().manual_seed(13)
    q = torch.randn(cu[-1], 2, 64, generator=g)
    q[::2, :, 0] = 8.0                          # every other row: rise * 8 / 8
    q = q.to(dt).cuda()
    lse = torch.empty(cu[-1], 2, device="cuda")
    out = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld,
                                torch.from_numpy(cu.astype(np.int32)).cuda(), lse=lse)
    kernels.check_device_status()
    ref, mag, l_ref = paged.attention(_np(q), cache.k_ref, cache.v_ref, cache.table, lengths, cu,
                                      scale=0.125)
    u, score = U[dt], (1 + rise / 10) * 2.0 ** -13
    tol = u * np.abs(ref) + (u + 2 * score) * mag
    if dt is torch.float16:
        tol = tol + max(lengths) * 2.0 ** -25 * np.abs(cache.v_ref).max()
    assert (np.abs(_np(out) - ref) <= tol).all()
    assert (np.abs(_np(lse) - l_ref) <= score + 2.0 ** -20 * np.abs(l_ref)).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,hq,kv,page,softcap,window,alibi,prefix,pad", [
    (64, 4, 2, 16, 0, 0, False, None, 0), (128, 3, 1, 64, 0, 0, False, None, 30),
    (64, 2, 1, 256, 20.0, 60, True, None, 0), (128, 4, 4, 16, 0, 100, True, None, 60),
    (64, 5, 1, 32, 0, 0, True, [150, 0, 60], 40), (128, 2, 2, 128, 10.0, 0, False, [70, 280, 0], 0),
    (128, 8, 1, 32, 5.0, 33, False, None, 20)])
def test_values_that_are_not_finite_reach_only_their_readers(cuda, dtype, dim, hq, kv, page, softcap,
                                                             window, alibi, prefix, pad):
    """An infinity or a NaN in single columns of values that some rows of a block see and
    others do not: in front of a row, behind its window, ahead of it within a prefix,
    and before tokens that have no position.  The columns of rows that see one are not
    finite; everything else is what it is with zeros in their place."""
    from hybrid_llm_b200 import kernels
    dt = DT[dtype]
    new, context = [170, 40, 30], [30, 260, -12]
    lengths = [a + b for a, b in zip(new, context)]
    cache = Cache(lengths, kv, dim, page, dt, seed=72 + dim, pad=pad)
    cu = np.concatenate([[0], np.cumsum(new)])
    spots = [(0, 77, 3, float("nan")), (0, 78, dim - 1, float("inf")), (0, 198, 8, -float("inf")),
             (1, 250, 17, float("inf")), (1, 280, 40, float("nan")), (2, 0, 0, float("nan")),
             (2, 17, dim - 2, float("inf"))]
    see = np.zeros((cu[-1], dim), bool)      # columns that a row's keys make not finite
    seq, pos = paged.positions(cu, lengths, cu[-1])
    for b, key, col, what in spots:
        at = cache.table[b, key // page], slice(None), key % page, col
        cache.vd[at] = what
        cache.v_ref[at] = 0.0
        seen = (seq == b) & (pos >= 0) & ((key <= pos) & ((window == 0) | (pos - key < window)))
        if prefix is not None:
            seen |= (seq == b) & (pos >= 0) & (key < prefix[b])
        see[seen, col] = True
    g = torch.Generator().manual_seed(14)
    q = torch.randn(cu[-1], hq, dim, generator=g).to(dt).cuda()
    slopes = (torch.rand(hq, generator=g) * 0.2).cuda() if alibi else None
    pre = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    lse = torch.empty(cu[-1], hq, device="cuda")
    out = kernels.paged_prefill(q, cache.kd, cache.vd, cache.td, cache.ld,
                                torch.from_numpy(cu.astype(np.int32)).cuda(), softcap=softcap,
                                window=window, slopes=slopes, prefix=pre, lse=lse)
    kernels.check_device_status()
    there = torch.from_numpy(see).cuda()[:, None, :].expand(out.shape)
    assert see.any() and not see.all(0).any()
    assert not out[there].isfinite().any()
    ref, _, _ = paged.attention(_np(q), cache.k_ref, cache.v_ref, cache.table, cache.lengths, cu,
                                scale=dim ** -0.5, softcap=softcap, window=window, prefix=prefix,
                                slopes=None if slopes is None else _np(slopes))
    out = torch.where(there, torch.from_numpy(ref).cuda().to(dt), out)
    _check(out, lse, cache, q, cu, dt, softcap=softcap, window=window, prefix=prefix,
           slopes=None if slopes is None else _np(slopes))


def test_tables_without_columns(cuda):
    """No row has a page yet: outputs are zero, an append has nowhere to store."""
    from hybrid_llm_b200 import kernels
    cache = Cache([40, 9], 2, 64, 16, torch.bfloat16, seed=50)
    x = torch.randn(2, 8, 64, device="cuda").bfloat16()
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    cu = torch.arange(3, dtype=torch.int32, device="cuda")
    table, none = cache.td[:, :0], torch.zeros_like(cache.ld)
    before = cache.kd.clone()
    for lengths in (none, cache.ld):  # attention counts what the table holds
        for out in (kernels.paged_decode(q, cache.kd, cache.vd, table, lengths),
                    kernels.paged_prefill(q, cache.kd, cache.vd, table, lengths, cu)):
            assert (out == 0).all()
    for packed in (None, cu):
        assert (kernels.paged_append(q, k, v, cache.kd, cache.vd, table, none, cu_q=packed) == 0).all()
    kernels.check_device_status()
    kernels.paged_append(q, k, v, cache.kd, cache.vd, table, cache.ld)
    with pytest.raises(RuntimeError, match="invalid argument"):
        kernels.check_device_status()
    assert torch.equal(cache.kd.view(torch.int16), before.view(torch.int16))
