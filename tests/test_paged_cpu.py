"""CPU: host-side argument checks of the paged cache and of beam search's selection through the C ABI (they come
before any CUDA call), and the oracle's own invariants."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from cudallm_b200 import abi, paged
from oracle import paged64 as R

FAKE = 1 << 20  # an aligned address that nothing reads: every call here is refused


@pytest.fixture(autouse=True)
def _lib(native_lib):
    return native_lib


def _struct(name, **fields):
    a = abi.struct(name)()
    a.struct_size = ctypes.sizeof(a)
    for k, v in fields.items():
        setattr(a, k, v)
    return a


def _pages(**over):
    f = dict(kv_dtype=0, n_layers=2, n_pages=8, n_kv_heads=2, page_size=16, head_dim=64, k=FAKE, v=FAKE, layer_stride=16384, page_stride=2048,
             head_stride=1024, token_stride=64)
    return _struct("cudallm_pages", **{**f, **over})


def _attend(**over):
    f = dict(layer=0, x_dtype=0, n_seq=2, n_heads=4, table_width=3, window=0, scale=0.125, q=FAKE, q_seq_stride=256, q_head_stride=64, tables=FAKE,
             table_stride=3, lens=FAKE, out=2 * FAKE, workspace=FAKE, workspace_bytes=1 << 40)
    return _struct("cudallm_attend_args", **{**f, **over})


def _append(**over):
    f = dict(layer=0, x_dtype=0, n_tokens=2, n_heads=4, n_rows=2, table_width=3, rotary=64, interleaved=0, factor=1.0, q=FAKE, k=FAKE, v=FAKE,
             q_token_stride=256, q_head_stride=64, inv_freq=FAKE, positions=FAKE, tables=FAKE, table_stride=3, q_out=FAKE, out_token_stride=256,
             out_head_stride=64)
    return _struct("cudallm_append_args", **{**f, **over})


def _fork(**over):
    f = dict(n_rows=2, n_out=2, table_width=3, room=1, tables=FAKE, table_stride=3, lens=2 * FAKE, refs=3 * FAKE, parents=4 * FAKE, tables_out=5 * FAKE,
             table_out_stride=3, lens_out=6 * FAKE, refs_out=7 * FAKE, missing=8 * FAKE, workspace=9 * FAKE, workspace_bytes=1 << 40)
    return _struct("cudallm_fork_args", **{**f, **over})


def _compact(**over):
    f = dict(n_rows=2, table_width=3, tables=FAKE, table_stride=3, refs=3 * FAKE, tables_out=5 * FAKE, table_out_stride=3, refs_out=7 * FAKE,
             live=8 * FAKE, workspace=9 * FAKE, workspace_bytes=1 << 40)
    return _struct("cudallm_compact_args", **{**f, **over})


def _beam(**over):
    f = dict(x_dtype=0, n_groups=2, beams=4, keep=4, vocab=100, eos=0, logits=FAKE, row_stride=100, scores=FAKE, out_scores=FAKE, out_parents=FAKE,
             out_tokens=FAKE, workspace=FAKE, workspace_bytes=1 << 40)
    return _struct("cudallm_beam_args", **{**f, **over})


def _refused(lib, fn, *structs) -> bool:
    return getattr(lib, fn)(*(None if s is None else ctypes.byref(s) for s in structs), None) == 1


@pytest.mark.parametrize("over", [dict(struct_size=8), dict(kv_dtype=2), dict(n_pages=0), dict(page_size=-1), dict(head_dim=60), dict(head_dim=264), dict(k=None),
                                  dict(v=FAKE + 8), dict(page_stride=1024), dict(token_stride=60), dict(token_stride=68), dict(layer_stride=-16384), dict(head_stride=0)],
                         ids=str)
def test_pools_that_are_refused(native_lib, over):
    for fn, args in (("cudallm_paged_attend", _attend()), ("cudallm_paged_append", _append()), ("cudallm_paged_fork", _fork()),
                     ("cudallm_paged_compact", _compact())):
        assert _refused(native_lib, fn, _pages(**over), args), fn
        assert _refused(native_lib, fn, None, args) and _refused(native_lib, fn, _pages(), None)


@pytest.mark.parametrize("over", [dict(struct_size=0), dict(layer=2), dict(layer=-1), dict(x_dtype=3), dict(n_seq=-1), dict(n_seq=65537), dict(n_heads=0), dict(n_heads=5),
                                  dict(window=-1), dict(scale=float("inf")), dict(q=None), dict(q=FAKE + 2), dict(lens=None), dict(out=None), dict(tables=None),
                                  dict(table_stride=2), dict(table_width=-1), dict(table_width=1 << 28, table_stride=1 << 28), dict(out=FAKE + 1024), dict(q_seq_stride=-1),
                                  dict(workspace=None), dict(workspace_bytes=100), dict(workspace=FAKE + 16), dict(lse=FAKE + 2)], ids=str)
def test_attend_refusals(native_lib, over):
    assert _refused(native_lib, "cudallm_paged_attend", _pages(), _attend(**over))


@pytest.mark.parametrize("over", [dict(struct_size=0), dict(layer=9), dict(x_dtype=-1), dict(n_tokens=-1), dict(n_heads=0), dict(rotary=3), dict(rotary=66), dict(rotary=-2),
                                  dict(inv_freq=None), dict(k=None), dict(v=None), dict(positions=None), dict(q_out=None), dict(factor=float("nan")),
                                  dict(q_out=FAKE + 4), dict(out_head_stride=32), dict(out_token_stride=0), dict(k_head_stride=-8), dict(tables=None),
                                  dict(out_token_stride=192), dict(rows=FAKE + 1)], ids=str)
def test_append_refusals(native_lib, over):
    assert _refused(native_lib, "cudallm_paged_append", _pages(), _append(**over))


@pytest.mark.parametrize("over", [dict(out=6 * FAKE - 2044), dict(out=6 * FAKE), dict(out=5 * FAKE + 20), dict(lse=FAKE + 2044), dict(lse=2 * FAKE), dict(lse=5 * FAKE - 28), dict(lse=6 * FAKE + 4),
                                  dict(lse=2 * FAKE + 2044)], ids=str)
def test_attend_refuses_outputs_over_inputs_or_each_other(native_lib, over):
    apart = dict(q=FAKE, out=2 * FAKE, lse=3 * FAKE, tables=5 * FAKE, lens=6 * FAKE)
    assert _refused(native_lib, "cudallm_paged_attend", _pages(), _attend(**{**apart, **over}))
    assert b"overlap" in native_lib.cudallm_last_error()
    assert _refused(native_lib, "cudallm_paged_attend", _pages(), _attend(**apart, workspace_bytes=8))  # as they are, only the workspace is refused
    assert b"workspace" in native_lib.cudallm_last_error()


@pytest.mark.parametrize("over", [dict(positions=2 * FAKE + 2044), dict(rows=2 * FAKE - 4), dict(tables=2 * FAKE + 1024), dict(inv_freq=2 * FAKE - 124)], ids=str)
def test_append_refuses_outputs_over_indexes(native_lib, over):
    apart = dict(q=FAKE, q_out=2 * FAKE, k=3 * FAKE, v=4 * FAKE, positions=5 * FAKE, rows=6 * FAKE, tables=7 * FAKE, inv_freq=8 * FAKE, factor=float("nan"), k_token_stride=128,
                 k_head_stride=64, v_token_stride=128, v_head_stride=64)
    assert _refused(native_lib, "cudallm_paged_append", _pages(), _append(**{**apart, **over}))
    assert b"overlap" in native_lib.cudallm_last_error()
    assert _refused(native_lib, "cudallm_paged_append", _pages(), _append(**apart))
    assert b"factor" in native_lib.cudallm_last_error()


def test_append_refuses_outputs_over_the_keys_or_values(native_lib):
    """Layouts of q_out, k and v around each other, in one buffer: refused exactly where a head of q_out shares a byte with a head of k or v, for equal
    token strides; for others wherever they share one. (factor is not a number, so that every call is refused by one check or the other.)"""
    rng = np.random.default_rng(0)
    counts = {True: 0, False: 0}
    for i in range(6000):
        T, H, KV, hd = int(rng.integers(1, 5)), int(rng.integers(1, 4)), int(rng.integers(1, 4)), 8
        hs = [int(rng.choice([8, 9, 12, 16, 24, 40, 41])) for _ in range(3)]
        ts = [int(rng.choice([8, 24, 33, 48, 64, 72, 100, 120]))] * 3 if i % 3 else [int(rng.choice([24, 48, 64, 100])) for _ in range(3)]
        if i % 5 == 0:
            hs = [hs[0]] * 3
        at = [0, *(int(rng.integers(-200, 200)) for _ in range(2))]
        base = FAKE + 4096
        assert _refused(native_lib, "cudallm_paged_append", _pages(n_kv_heads=KV, head_dim=hd, page_size=1, token_stride=8, head_stride=8, page_stride=KV * 8, layer_stride=KV * 64),
                        _append(n_tokens=T, n_rows=T, n_heads=H, rotary=8, factor=float("nan"), q=4 * FAKE, q_token_stride=64, q_head_stride=8,
                                q_out=base, out_token_stride=ts[0], out_head_stride=hs[0], k=base + 4 * at[1], k_token_stride=ts[1], k_head_stride=hs[1],
                                v=base + 4 * at[2], v_token_stride=ts[2], v_head_stride=hs[2]))
        message = native_lib.cudallm_last_error()
        sets = [{a + t * x + h * y + e for t in range(T) for h in range(n) for e in range(hd)} for a, x, y, n in zip(at, ts, hs, (H, KV, KV))]
        meets = bool(sets[0] & sets[1] or sets[0] & sets[2])
        if b"heads of q_out must not overlap" in message:
            continue
        refused = b"must not overlap k or v" in message
        assert refused or b"factor" in message, message
        assert refused or not meets, (T, H, KV, hs, ts, at)
        if len(set(ts)) == 1:
            assert refused == meets, (T, H, KV, hs, ts, at)
            counts[meets] += 1
    assert min(counts.values()) > 300, counts


@pytest.mark.parametrize("over", [dict(struct_size=0), dict(n_rows=-1), dict(n_out=65537), dict(room=-1), dict(tables=None), dict(lens=None), dict(refs=None),
                                  dict(parents=None), dict(tables_out=FAKE), dict(tables_out=FAKE + 20), dict(refs_out=3 * FAKE), dict(missing=3 * FAKE + 28),
                                  dict(lens_out=5 * FAKE + 4), dict(missing=None), dict(workspace_bytes=0), dict(table_out_stride=1)], ids=str)
def test_fork_refusals(native_lib, over):
    assert _refused(native_lib, "cudallm_paged_fork", _pages(), _fork(**over))


@pytest.mark.parametrize("over", [dict(struct_size=0), dict(n_rows=-1), dict(tables=None), dict(refs=None), dict(refs_out=3 * FAKE), dict(live=None), dict(live=7 * FAKE),
                                  dict(tables_out=FAKE + 8), dict(workspace=None), dict(table_stride=0)], ids=str)
def test_compact_refusals(native_lib, over):
    assert _refused(native_lib, "cudallm_paged_compact", _pages(), _compact(**over))


@pytest.mark.parametrize("over", [dict(struct_size=0), dict(x_dtype=3), dict(n_groups=-1), dict(n_groups=1 << 20), dict(beams=0), dict(beams=65), dict(keep=0), dict(keep=65),
                                  dict(vocab=0), dict(beams=1, vocab=3, row_stride=3), dict(logits=None), dict(logits=FAKE + 2), dict(scores=None), dict(out_tokens=None),
                                  dict(row_stride=99), dict(finished=FAKE, eos=100), dict(finished=FAKE, eos=-1), dict(workspace_bytes=8)], ids=str)
def test_beam_refusals(native_lib, over):
    assert _refused(native_lib, "cudallm_beam_select", _beam(**over))


APART = dict(logits=FAKE, scores=2 * FAKE, finished=3 * FAKE, out_scores=4 * FAKE, out_parents=5 * FAKE, out_tokens=6 * FAKE, workspace=7 * FAKE)


@pytest.mark.parametrize("over", [dict(out_scores=2 * FAKE + 4), dict(out_scores=2 * FAKE, keep=5), dict(out_scores=2 * FAKE, keep=3), dict(out_parents=2 * FAKE), dict(out_tokens=2 * FAKE + 28),
                                  dict(out_parents=3 * FAKE - 28), dict(out_tokens=FAKE + 400), dict(out_scores=FAKE + 3196), dict(out_tokens=5 * FAKE + 16), dict(out_parents=4 * FAKE),
                                  dict(row_stride=107, out_parents=FAKE + 400), dict(row_stride=108, out_parents=FAKE + 432 * 7 + 396), dict(row_stride=0, out_scores=FAKE + 396)],
                         ids=str)
def test_beam_refuses_overlaps(native_lib, over):
    assert _refused(native_lib, "cudallm_beam_select", _beam(**{**APART, **over}))
    assert b"overlap" in native_lib.cudallm_last_error()


@pytest.mark.parametrize("over", [dict(), dict(out_scores=2 * FAKE), dict(out_scores=2 * FAKE + 32), dict(out_scores=FAKE + 3200), dict(row_stride=108, out_parents=FAKE + 400),
                                  dict(row_stride=108, out_parents=FAKE + 432 * 7 + 400), dict(row_stride=0, out_scores=FAKE + 400), dict(finished=None, out_tokens=3 * FAKE)], ids=str)
def test_beam_takes_what_lies_apart(native_lib, over):
    """The workspace is too small, so that these are refused as well, after the check for overlaps."""
    assert _refused(native_lib, "cudallm_beam_select", _beam(**{**APART, **over, "workspace_bytes": 8}))
    assert b"workspace" in native_lib.cudallm_last_error()


def test_messages_and_workspace_sizes(native_lib):
    assert _refused(native_lib, "cudallm_paged_attend", _pages(), _attend(layer=7))
    assert b"layer" in native_lib.cudallm_last_error()
    assert native_lib.cudallm_attend_workspace_bytes() > 0
    assert native_lib.cudallm_pages_workspace_bytes(1000, 64) > 4000
    assert native_lib.cudallm_pages_workspace_bytes(0, 64) == 0 and native_lib.cudallm_pages_workspace_bytes(8, 1 << 20) == 0
    assert native_lib.cudallm_beam_workspace_bytes(64, 128256, 16) > 64 * 16 * 8 and native_lib.cudallm_beam_workspace_bytes(4, 100, 65) == 0


def test_a_graph_keeps_its_workspace_whichever_device_is_current(monkeypatch):
    """Calls for device 1 while its stream is captured and device 0 is current: each workspace is the graph's own. Otherwise the stream's is kept."""
    now, capturing = [0], [1]
    monkeypatch.setattr(paged, "_current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "set_device", lambda i: now.__setitem__(0, i))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] in capturing)
    monkeypatch.setattr(paged._Workspaces, "_new", lambda self, size: torch.empty(size, dtype=torch.uint8))
    spaces = paged._Workspaces(torch.device("cuda", 1))
    for current in (0, 1):
        now[0] = current
        a, b = spaces.get(7, 100), spaces.get(7, 100)
        assert a is not b and not spaces.by_stream and now[0] == current
    capturing[0] = 0  # a capture on another device does not matter
    a = spaces.get(7, 100)
    assert a is spaces.get(7, 100) and spaces.by_stream[7] is a


def test_tensors_off_the_gpu_are_refused():
    k = torch.zeros((1, 2, 1, 8, 64), dtype=torch.float16)
    with pytest.raises(paged.CudaLLMError):
        paged.PagedCache(k, k)
    with pytest.raises(paged.CudaLLMError):
        paged.Rope(torch.zeros(4))
    with pytest.raises(paged.CudaLLMError):
        paged.Rope.make(63)
    with pytest.raises(paged.CudaLLMError):
        paged.beam_select(torch.zeros((2, 5)), torch.zeros((1, 2)), keep=1)


def test_oracle_fork_keeps_references_and_contents():
    """Walks of forks on random parents: references equal the tables' entries, and every row's tokens are its ancestor's."""
    rng = np.random.default_rng(0)
    page, pages = 4, 60
    content = np.full((pages, page), -1)
    tables, lens, refs = np.full((1, 12), -1), np.array([0]), np.zeros(pages, np.int64)
    texts = [[]]
    for step in range(25):
        parents = rng.integers(0, len(lens), 4)
        tables, lens, refs, missing, copies = R.fork_ref(tables, lens, refs, parents, page, 1)
        assert missing == 0
        for src, dst, n in copies:
            content[dst, :n] = content[src, :n]
        texts = [list(texts[p]) for p in parents]
        for r in range(4):
            content[tables[r][lens[r] // page], lens[r] % page] = 100 * step + r
            texts[r].append(100 * step + r)
            lens[r] += 1
        assert np.array_equal(np.bincount(tables[tables >= 0], minlength=pages), refs)
        for r in range(4):
            assert [content[tables[r][t // page], t % page] for t in range(lens[r])] == texts[r]
