"""CPU checks of the paged cache and of beam selection: refusals at the Python and at the C boundary, and the oracle itself."""

import ctypes

import pytest
import torch

import paged_oracle
import selective_oracle as oracle
from selective_attention_b200 import _lib, beams, kernels, mixers, paged


def _cpu_tables(rows=3, num_pages=8, page=16, max_pages=4, heads=2):
    return paged.begin_tables(rows, num_pages, page, max_pages, heads, device="cpu")


def test_tables_begin_empty():
    t = _cpu_tables()
    assert t["block_tables"].shape == (3, 4) and (t["block_tables"] == -1).all() and t["lengths"].sum() == 0
    assert t["free_pages"].tolist() == list(range(7, -1, -1)) and t["free_count"].item() == 8
    cache = paged.begin_pages(t, 64)
    assert cache["k"].shape == (8, 2, 16, 64) and cache["k"].dtype == torch.bfloat16 and cache["selected"].shape == (3, 1, 64)
    slot = mixers.SelectiveAttentionSlot(2, 64, per_head=True)
    assert slot.begin_pages(t, 128)["selected"].shape == (3, 2, 64)


@pytest.mark.parametrize("kw", [dict(page=24), dict(page=8), dict(rows=0), dict(rows=4097), dict(num_pages=0), dict(max_pages=0),
                                dict(heads=0), dict(heads=257)])
def test_tables_that_are_refused(kw):
    with pytest.raises(ValueError):
        _cpu_tables(**kw)


def test_calls_on_cpu_tensors_are_refused():
    t = _cpu_tables()
    counts = torch.ones(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.append_tokens(t, counts, 3)
    with pytest.raises(ValueError, match="CUDA"):
        paged.reorder_rows(t, counts)
    cache, x = paged.begin_pages(t, 64), torch.zeros(3, 2, 64)
    step = {"_plan": None}                                         # a step is made on the GPU
    with pytest.raises(TypeError):
        paged.paged_attention(cache, t, step, x, x, x)
    with pytest.raises(ValueError, match="exempt"):
        paged.paged_attention(cache, t, step, x, x, x, exempt=0)
    with pytest.raises(ValueError, match="CUDA"):
        paged.move_rows(cache, {"tables": t, "copies": torch.zeros(3, 2, dtype=torch.int32), "_work": counts})
    with pytest.raises(ValueError, match="CUDA"):
        beams.beam_select(torch.zeros(1, 2, 10), torch.zeros(1, 2), 2)
    with pytest.raises(ValueError, match="logits must be"):
        beams.beam_select(torch.zeros(2, 10), torch.zeros(1, 2), 2)
    with pytest.raises(ValueError, match="head_dim"):
        paged.begin_pages(t, 32)
    with pytest.raises(ValueError, match="heads"):
        mixers.SelectiveAttentionSlot(4, 64).begin_pages(t, 64)
    with pytest.raises(ValueError, match="selectors"):
        mixers.SelectiveAttentionSlot(2, 64, per_head=True).attend_pages(x, x, x, cache, t, step)


def _c_tables(**kw):
    t = _lib.PageTables()
    t.struct_bytes = ctypes.sizeof(_lib.PageTables)
    t.rows, t.max_pages, t.num_pages, t.page_size, t.heads = 4, 8, 32, 16, 2
    t.block_tables = t.lengths = t.free_pages = t.free_count = t.page_refs = 4096
    for name, value in kw.items():
        setattr(t, name, value)
    return t


@pytest.mark.parametrize("kw,status", [(dict(struct_bytes=4), 1), (dict(rows=0), 1), (dict(rows=4097), 2), (dict(page_size=48), 2),
                                       (dict(page_size=512), 2), (dict(heads=300), 2), (dict(lengths=None), 1), (dict(page_refs=4098), 3),
                                       (dict(num_pages=1 << 28), 7)])
def test_bad_tables_are_refused_before_any_launch(kw, status):
    lib, t = _lib.load(), _c_tables(**kw)
    assert lib.sa_page_append(ctypes.byref(t), 4096, 4, 64, 4, 4096, 4096, 4096, 4096, None) == status
    assert lib.sa_page_reorder(ctypes.byref(t), 4096, 4096, 4096, None) == status
    assert lib.sa_page_move(ctypes.byref(t), 4096, 4096, 1, 64, 4096, 4096, 4096, None) == status


def test_bad_steps_are_refused_before_any_launch():
    lib, t = _lib.load(), _c_tables()
    call = lambda **kw: lib.sa_page_append(*[{**dict(t=ctypes.byref(t), counts=4096, total=4, length=64, count=4, starts=4096, cached=4096,  # noqa: E731
                                                    slots=4096, work=4096, stream=None), **kw}[n]
                                             for n in ("t", "counts", "total", "length", "count", "starts", "cached", "slots", "work", "stream")])
    assert call(counts=None) == 1 and call(total=-1) == 1 and call(length=0) == 1 and call(count=0) == 1 and call(slots=None) == 1
    assert call(work=4104) == 3 and call(slots=4100) == 3 and call(total=(1 << 30) + 1) == 7
    assert lib.sa_page_step_words(0, 4, 2) == 0 and lib.sa_page_step_words(4, -1, 2) == 0 and lib.sa_page_step_words(4, 4, 2) > 0
    assert lib.sa_page_reorder_words(4097, 1, 1) == 0


def test_bad_attention_is_refused_before_any_launch():
    lib, t = _lib.load(), _c_tables()

    def status(**kw):
        p = _lib.PagedAttention()
        p.struct_bytes = ctypes.sizeof(_lib.PagedAttention)
        p.tables = ctypes.pointer(t)
        p.groups, p.head_dim, p.exempt, p.total, p.max_length, p.max_count = 1, 64, 1, 4, 64, 4
        for name in ("query_start", "cached", "slots", "work", "k_pages", "v_pages", "selected", "q", "k", "v", "y", "workspace"):
            setattr(p, name, 4096)
        for name in ("q_stride", "k_stride", "v_stride"):
            getattr(p, name)[:] = [128, 64]
        p.workspace_bytes = 0
        for name, value in kw.items():
            if name.endswith("stride"):
                getattr(p, name)[:] = value
            else:
                setattr(p, name, value)
        return lib.sa_paged_run(ctypes.byref(p)), lib.sa_paged_workspace_bytes(ctypes.byref(p))

    assert status()[0] == 4 and status()[1] > 0                    # workspace_bytes 0
    assert status(struct_bytes=8) == (1, 0) and status(exempt=0)[0] == 1 and status(total=0)[0] == 1 and status(max_length=129)[0] == 1
    assert status(head_dim=32)[0] == 2 and status(groups=3)[0] == 2 and status(q=None)[0] == 1 and status(y=None)[0] == 1
    assert status(k_pages=4104)[0] == 3 and status(q_stride=[128, 68])[0] == 3 and status(v_stride=[128, 0])[0] == 3 and status(workspace=4112)[0] == 3


def test_attention_takes_rows_from_the_plan_alone():
    """What the plan holds already need not be given a second time: a call without it gets as far as its workspace."""
    lib, t = _lib.load(), _c_tables()
    p = _lib.PagedAttention()
    p.struct_bytes = ctypes.sizeof(_lib.PagedAttention)
    p.tables = ctypes.pointer(t)
    p.groups, p.head_dim, p.exempt, p.total, p.max_length, p.max_count = 1, 64, 1, 4, 64, 4
    for name in ("slots", "work", "k_pages", "v_pages", "selected", "q", "k", "v", "y", "workspace"):
        setattr(p, name, 4096)
    for name in ("q_stride", "k_stride", "v_stride"):
        getattr(p, name)[:] = [128, 64]
    assert lib.sa_paged_run(ctypes.byref(p)) == 4                  # workspace_bytes 0
    for name in ("slots", "work"):
        setattr(p, name, None)
        assert lib.sa_paged_run(ctypes.byref(p)) == 1
        setattr(p, name, 4096)


@pytest.mark.parametrize("exempt", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 10 ** 30])
def test_exemptions_beyond_32_bits_exempt_everything(exempt):
    slot = mixers.SelectiveAttentionSlot(2, 64, exempt=exempt)
    assert ctypes.c_int32(slot.exempt).value == slot.exempt == 2 ** 31 - 1
    q = torch.randn(1, 2, 9, 16)
    assert kernels.selective_logits(q, q, exempt)[1].abs().max() == 0


def test_bad_selections_are_refused_before_any_launch():
    lib = _lib.load()

    def status(**kw):
        p = _lib.Beam()
        p.struct_bytes = ctypes.sizeof(_lib.Beam)
        p.dtype, p.groups, p.beams, p.vocab, p.width, p.group_stride, p.beam_stride = 0, 2, 4, 100, 4, 400, 100
        for name in ("logits", "scores", "out_scores", "out_rows", "out_tokens", "workspace"):
            setattr(p, name, 4096)
        for name, value in kw.items():
            setattr(p, name, value)
        return lib.sa_beam_select(ctypes.byref(p))

    assert status() == 4 and status(struct_bytes=0) == 1 and status(dtype=3) == 1 and status(width=0) == 1 and status(width=33) == 2
    assert status(beams=257) == 2 and status(vocab=1, beams=2, width=4) == 2 and status(logits=None) == 1 and status(logits=4098) == 3
    assert status(groups=1 << 20) == 7


def test_attention_oracle_equals_the_dense_one():
    """A row's chunks through the paged oracle, against the whole sequence through the dense one."""
    gen = torch.Generator().manual_seed(3)
    for per_head in (False, True):
        q, k, v = (torch.randn(300, 3, 16, generator=gen, dtype=torch.float64) for _ in range(3))
        split = (lambda x: x.permute(1, 0, 2)[:, None]) if per_head else (lambda x: x.permute(1, 0, 2)[None])
        z, total = oracle.history_logits(split(q), split(k), exempt=2)
        want = (z.double().softmax(-1) @ split(v)).reshape(3, 300, 16).permute(1, 0, 2)
        history, at = torch.zeros(3 if per_head else 1, 0), 0
        for n in (1, 130, 1, 168):
            y, history, off, _ = paged_oracle.attend(q[at:at + n], k[:at + n], v[:at + n], history, at, 2, per_head)
            torch.testing.assert_close(y, want[at:at + n].double(), atol=1e-4, rtol=1e-4)      # the dense one is in 32 bits
            assert (off >= 2.0 ** -8 * y.abs()).all()
            at += n
        torch.testing.assert_close(history, total.reshape(history.shape).double(), atol=1e-3, rtol=1e-4)


def test_table_oracle_keeps_its_books():
    t = paged_oracle.Tables(4, 12, 16, 6)
    t.append([20, 0, 33, 1], 54)
    t.reorder([2, 2, 0, 3])
    t.append([5, 30, 1, 1], 37)
    t.reorder([-1, 1, 9, 1])
    held = [p for blocks in t.blocks for p in blocks]
    assert all(t.refs[p] == held.count(p) for p in range(12)) and sorted(t.free + sorted(set(held))) == list(range(12))
    assert t.lengths[0] == t.lengths[2] == 0 and t.lengths[1] == t.lengths[3] == 63
