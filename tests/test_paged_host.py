"""CPU: the paged cache's page bookkeeping, and what the C entry points refuse
before they touch a device."""
import ctypes as C

import pytest
import torch

from hybrid_llm_b200 import _native, kernels
from hybrid_llm_b200.state import PagedKVCache

POINTERS = ("q k v q_norm k_norm inv_freq k_pages v_pages table lengths cu_q prefix slopes out lse "
            "scratch dev_status").split()


class Args(C.Structure):
    """llmyb_paged_args of include/llmyb.h."""
    _fields_ = ([(n, C.c_void_p) for n in POINTERS]
                + [(n, C.c_int64) for n in (
                    "q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride",
                    "v_token_stride", "v_head_stride", "out_token_stride", "out_head_stride",
                    "page_stride", "head_stride", "row_stride", "table_stride")]
                + [(n, C.c_int32) for n in (
                    "n_tokens", "batch", "q_heads", "kv_heads", "head_dim", "fp16", "num_pages",
                    "page_size", "table_width", "window", "rope_half", "interleaved")]
                + [(n, C.c_float) for n in ("scale", "softcap", "eps")] + [("reserved", C.c_int32)])


def _args(**over):
    """A block that every call would accept (the addresses are never followed)."""
    a = Args()
    for n in POINTERS:
        if n not in ("prefix", "lse", "slopes"):
            setattr(a, n, 1 << 20)
    for n, t in Args._fields_:
        if t is C.c_int64:
            setattr(a, n, 64)
    a.n_tokens = a.batch = 4
    a.q_heads, a.kv_heads, a.head_dim, a.num_pages, a.page_size, a.table_width = 4, 2, 64, 8, 16, 4
    a.scale, a.eps = 0.125, 1e-6
    for n, v in over.items():
        setattr(a, n, v)
    return a


def _status(entry, a):
    return getattr(_native.lib(), entry)(C.byref(a), None)


APPEND, DECODE, PREFILL = ("llmyb_paged_append", "llmyb_paged_decode", "llmyb_paged_prefill")


@pytest.mark.parametrize("entry", [APPEND, DECODE, PREFILL])
def test_common_refusals(entry):
    for over, status in (
            (dict(n_tokens=-1), _native.LLMYB_EINVAL), (dict(batch=-1), _native.LLMYB_EINVAL),
            (dict(q_heads=0), _native.LLMYB_EINVAL), (dict(kv_heads=0), _native.LLMYB_EINVAL),
            (dict(num_pages=-1), _native.LLMYB_EINVAL), (dict(num_pages=0), _native.LLMYB_EINVAL),
            (dict(table_width=-1), _native.LLMYB_EINVAL),
            *((({n: None}), _native.LLMYB_EINVAL)
              for n in ("q", "k_pages", "v_pages", "table", "lengths", "out")),
            (dict(page_size=24), _native.LLMYB_EUNSUPPORTED),
            (dict(page_size=0), _native.LLMYB_EUNSUPPORTED),
            (dict(head_dim=96), _native.LLMYB_EUNSUPPORTED),
            (dict(table_width=1 << 30), _native.LLMYB_EUNSUPPORTED),
            (dict(q=(1 << 20) + 8), _native.LLMYB_EUNSUPPORTED),
            (dict(out=(1 << 20) + 2), _native.LLMYB_EUNSUPPORTED),
            (dict(q_token_stride=65), _native.LLMYB_EUNSUPPORTED),
            (dict(out_head_stride=4), _native.LLMYB_EUNSUPPORTED),
            (dict(page_stride=100), _native.LLMYB_EUNSUPPORTED),
            (dict(row_stride=63), _native.LLMYB_EUNSUPPORTED)):
        assert _status(entry, _args(**over)) == status, over
    assert getattr(_native.lib(), entry)(None, None) == _native.LLMYB_EINVAL
    # nothing to do: no pointer is needed
    assert _status(entry, _args(n_tokens=0, batch=0, q=None, out=None, scratch=None)) == 0


def test_append_refusals():
    for over, status in (
            (dict(k=None), _native.LLMYB_EINVAL), (dict(v=None), _native.LLMYB_EINVAL),
            (dict(rope_half=8, inv_freq=None), _native.LLMYB_EINVAL),
            (dict(rope_half=-8), _native.LLMYB_EINVAL), (dict(eps=-1.0), _native.LLMYB_EINVAL),
            (dict(eps=float("nan")), _native.LLMYB_EINVAL),
            (dict(cu_q=None, n_tokens=5), _native.LLMYB_EINVAL),
            (dict(rope_half=12), _native.LLMYB_EUNSUPPORTED),
            (dict(rope_half=40), _native.LLMYB_EUNSUPPORTED),
            (dict(q_norm=(1 << 20) + 4), _native.LLMYB_EUNSUPPORTED),
            (dict(k_token_stride=4), _native.LLMYB_EUNSUPPORTED),
            (dict(v=(1 << 20) + 4), _native.LLMYB_EUNSUPPORTED)):
        assert _status(APPEND, _args(**over)) == status, over


@pytest.mark.parametrize("entry", [DECODE, PREFILL])
def test_attention_refusals(entry):
    for over in (dict(q_heads=3), dict(window=-1), dict(scale=0.0), dict(scale=-1.0),
                 dict(scale=float("nan")), dict(softcap=-1.0), dict(softcap=float("nan"))):
        assert _status(entry, _args(**over)) == _native.LLMYB_EINVAL, over
    assert _status(entry, _args(scratch=(1 << 20) + 4)) == _native.LLMYB_EUNSUPPORTED


def test_decode_and_prefill_refusals():
    assert _status(DECODE, _args(n_tokens=5)) == _native.LLMYB_EINVAL
    assert _status(DECODE, _args(scratch=None)) == _native.LLMYB_EINVAL
    assert _status(PREFILL, _args(cu_q=None)) == _native.LLMYB_EINVAL
    assert _status(PREFILL, _args(prefix=1 << 20, window=3)) == _native.LLMYB_EINVAL
    assert _status(PREFILL, _args(q_heads=260)) == _native.LLMYB_EUNSUPPORTED
    # 64 pages of 16 positions: units may be cut, so scratch is needed
    assert _status(PREFILL, _args(scratch=None, table_width=64)) == _native.LLMYB_EINVAL


def test_scratch_sizes():
    lib = _native.lib()
    assert lib.llmyb_paged_decode_scratch_bytes(3, 2, 64) == -1
    assert lib.llmyb_paged_decode_scratch_bytes(8, 2, 128) > 0
    assert lib.llmyb_paged_prefill_scratch_bytes(3, 2, 64, 10, 16) == -1
    assert lib.llmyb_paged_prefill_scratch_bytes(8, 2, 64, 8, 64) == 0      # 4 blocks of 128 keys
    assert lib.llmyb_paged_prefill_scratch_bytes(8, 2, 64, 9, 64) > 0


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    p = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: kernels.paged_append(x, x, x, p, p, t, n),
                 lambda: kernels.paged_decode(x, p, p, t, n),
                 lambda: kernels.paged_prefill(x, p, p, t, n, torch.tensor([0, 1], dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


# ------------------------------------------------------------------ the cache
def _cache(**over):
    return PagedKVCache(**{**dict(kv_heads=2, head_dim=64, batch=3, pages=8, page_size=16,
                                  device="cpu"), **over})


def _rows(c):
    return [[p for p in row if p >= 0] for row in c.block_table.tolist()]


def test_pages_follow_the_lengths():
    c = _cache(layers=2)
    assert len(c.k) == 2 and c.k[1].shape == (8, 2, 16, 64) and c.free_pages == 8
    assert c.extend([17, 0, 16]).tolist() == [0, 17, 17, 33]
    assert c.lengths.tolist() == [17, 0, 16]
    assert [len(r) for r in _rows(c)] == [2, 0, 1] and c.free_pages == 5
    assert c.extend([15, 1, 1]).tolist() == [0, 15, 16, 17]
    assert [len(r) for r in _rows(c)] == [2, 1, 2] and c.free_pages == 3
    held = sum(_rows(c), [])
    assert len(set(held)) == len(held)
    assert c.extend([0, 0, 0]).tolist() == [0, 0, 0, 0] and c.lengths.tolist() == [32, 1, 17]


def test_reserve_leaves_lengths_and_is_kept():
    c = _cache()
    c.reserve([40, 0, 0])
    assert c.lengths.tolist() == [0, 0, 0] and [len(r) for r in _rows(c)] == [3, 0, 0]
    before = _rows(c)
    c.extend([40, 0, 0])
    assert _rows(c) == before and c.free_pages == 5


def test_running_out_changes_nothing():
    c = _cache(max_pages=6)
    c.extend([48, 16, 16])
    state = _rows(c), c.lengths.tolist(), c.free_pages
    for tokens in ([0, 33, 17], [49, 0, 0]):  # 4 pages where 3 are free; 7 pages of one row
        with pytest.raises(RuntimeError):
            c.extend(tokens)
        assert (_rows(c), c.lengths.tolist(), c.free_pages) == state
    for tokens in ([1, 1], [1, 1, -1]):
        with pytest.raises(ValueError):
            c.extend(tokens)


def test_released_pages_come_back():
    c = _cache()
    c.extend([64, 64, 0])
    assert c.free_pages == 0
    c.release([1, 1])
    assert c.free_pages == 4 and c.lengths.tolist() == [64, 0, 0]
    assert [len(r) for r in _rows(c)] == [4, 0, 0]
    c.extend([0, 0, 64])
    held = sum(_rows(c), [])
    assert sorted(held) == list(range(8))


@pytest.mark.parametrize("over", [dict(page_size=24), dict(head_dim=96), dict(dtype=torch.float32),
                                  dict(pages=0), dict(batch=0), dict(layers=0), dict(kv_heads=0)])
def test_cache_refusals(over):
    with pytest.raises(ValueError):
        _cache(**over)


def test_lengths_counted_on_the_device_are_kept():
    """Steps that count the device's lengths up (a captured graph), told to the host
    by advance: extend goes on from them and reserve counts pages from them."""
    c = _cache(pages=16)
    c.extend([20, 5, 0])
    c.reserve([10, 10, 0])
    live = torch.tensor([1, 1, 0], dtype=torch.int32)
    for _ in range(10):
        c.lengths.add_(live)
    c.advance([10, 10, 0])
    assert c.lengths.tolist() == [30, 15, 0]
    assert c.extend([0, 7, 0]).tolist() == [0, 0, 7, 7]
    assert c.lengths.tolist() == [30, 22, 0] and [len(r) for r in _rows(c)] == [2, 2, 0]
    c.reserve([20, 0, 0])                            # positions 30 .. 49: two more pages
    assert [len(r) for r in _rows(c)] == [4, 2, 0]
    c.release([0])
    assert c.extend([3, 1, 0]).tolist() == [0, 3, 4, 4] and c.lengths.tolist() == [3, 23, 0]


def test_device_lengths_are_not_rewound():
    """Before advance is called, extend keeps what the device has counted."""
    c = _cache()
    c.extend([10, 0, 0])
    c.reserve([20, 0, 0])
    c.lengths[0] += 20
    c.extend([1, 0, 0])
    assert c.lengths.tolist() == [31, 0, 0]


def test_advance_refuses_what_has_no_page():
    c = _cache()
    c.extend([10, 3, 0])
    c.reserve([7, 0, 0])
    state = _rows(c), c.lengths.tolist(), c.free_pages
    for tokens in ([23, 0, 0], [0, 14, 0], [0, 0, 1]):
        with pytest.raises(RuntimeError, match="reserved"):
            c.advance(tokens)
    for tokens in ([1, 1], [1, -1, 0]):
        with pytest.raises(ValueError):
            c.advance(tokens)
    assert (_rows(c), c.lengths.tolist(), c.free_pages) == state
    c.advance([22, 13, 0])
    c.reserve([1, 1, 0])
    assert [len(r) for r in _rows(c)] == [3, 2, 0]


@pytest.mark.parametrize("entry", [DECODE, PREFILL])
def test_scores_that_fp32_does_not_hold_are_refused(entry):
    """A scale or a cap whose factors overflow or vanish: every score would be 0 or NaN."""
    inf = float("inf")
    for over in (dict(scale=inf), dict(scale=3e38), dict(scale=1e-40), dict(softcap=inf),
                 dict(softcap=3e38), dict(softcap=1e-39), dict(softcap=1e38), dict(scale=4.0, softcap=1e-38),
                 dict(scale=1e-30, softcap=1e9)):
        assert _status(entry, _args(**over)) == _native.LLMYB_EINVAL, over


@pytest.mark.parametrize("rows", [[0, 3], [-1], [1, -3], [99]])
def test_release_of_rows_that_are_none(rows):
    c = _cache()
    c.extend([20, 5, 16])
    state = _rows(c), c.lengths.tolist(), c.free_pages
    with pytest.raises(ValueError, match="released"):
        c.release(rows)
    assert (_rows(c), c.lengths.tolist(), c.free_pages) == state
    c.release([])
    c.release([2, 2, 0])
    assert c.lengths.tolist() == [0, 5, 0] and c.free_pages == 7
