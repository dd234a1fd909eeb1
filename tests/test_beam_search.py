"""Beam search over the paged cache (cudallm_b200/beam_search.py), where its operators run together.

  * with one beam it is greedy decoding: on the seeded full-size model it gives the ids of wasiqnauman/cudallm's
    ReferenceModel (golden_full_bf16_fp16);
  * with several it gives the hypotheses and scores of a plain beam search over the oracle model on the CPU, which
    recomputes every hypothesis from its first token. Scores are sums of at most 10 fp32 log-probabilities of magnitude
    below 16 from logits that agree to about 1e-4 (fp16 cache: a key or value may round the other way, 2^-11 of its
    size): 2e-3 is allowed, and the oracle's own choices must be further apart than that to be compared."""
from __future__ import annotations

import subprocess
import sys

import numpy as np
import pytest
import torch

import tiny_spec
from cudallm_b200 import format as fmt
from cudallm_b200.abi import CudaLLMError
from cudallm_b200.quantize import quantize_int4_groups, quantize_int8_rows

TOL = 2e-3


@pytest.fixture(scope="module")
def tiny(tmp_path_factory):
    paths = {}
    for dtype, code in (("bf16", fmt.WEIGHT_BF16), ("int8", fmt.WEIGHT_INT8), ("int4", fmt.WEIGHT_INT4)):
        paths[dtype] = tmp_path_factory.mktemp("beam") / f"{dtype}.cudallm"
        fmt.write_cudallm(paths[dtype], tiny_spec.header(code), tiny_spec.build_tensor_list(dtype, fmt, quantize_int8_rows, quantize_int4_groups))
    return paths


def _plain_search(path, prompt, beams, new_tokens, eos):
    """-> (hypotheses [(score, ids)] best first, the smallest gap between a candidate that was kept and its successor)."""
    from oracle.refmodel import RefModel
    model = RefModel(path, cache_dense=True)

    def log_probs(ids):
        model.reset()
        for t in ids:
            logits, _ = model.step(t)
        x = logits.double()
        return (x - torch.logsumexp(x, 0)).numpy()

    hyps, gap = [(0.0, [])], np.inf
    for _ in range(new_tokens):
        found = []
        for score, ids in hyps:
            if eos is not None and eos in ids:
                found.append((score, ids))
                continue
            lp = log_probs(prompt + ids)
            found += [(score + lp[t], ids + [int(t)]) for t in np.argsort(-lp)[:beams + 1]]
        found.sort(key=lambda f: -f[0])
        kept = found[:beams + 1]
        gap = min([gap] + [a[0] - b[0] for a, b in zip(kept, kept[1:])])
        hyps = found[:beams]
    return hyps, gap


PROMPTS = [tiny_spec.PROMPT, [5, 900, 31], [640] * 17]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, beams, page, eos", [("bf16", 3, 4, None), ("bf16", 4, 16, 777), ("int8", 2, 5, None), ("int4", 3, 1, None), ("bf16", 1, 64, None)])
def test_against_a_plain_search(native_lib, tiny, dtype, beams, page, eos):
    from cudallm_b200.beam_search import BeamSearch
    model = BeamSearch(tiny[dtype], rows=3 * beams, page_size=page)
    new = 7
    if eos is not None:  # a token that ends some of the hypotheses
        eos = _plain_search(tiny[dtype], PROMPTS[0], beams, 2, None)[0][1][1][0]
    found = model.search(PROMPTS, beams=beams, new_tokens=new, eos=eos)
    for prompt, got in zip(PROMPTS, found):
        want, gap = _plain_search(tiny[dtype], prompt, beams, new, eos)
        assert np.abs(np.array([g[0] for g in got]) - np.array([w[0] for w in want])).max() < TOL
        if gap > 2 * TOL:
            assert [g[1] for g in got] == [w[1] for w in want]


@pytest.mark.gpu
def test_one_beam_is_the_references_greedy_decoding(native_lib, model_path, golden):
    from cudallm_b200.beam_search import BeamSearch
    g = golden("full_bf16_fp16")
    path, digest = model_path("bf16")
    assert digest == str(g["digest"])
    model = BeamSearch(path, rows=1, max_seq_len=128)
    prompt, ids = [int(t) for t in g["prompt"]], [int(t) for t in g["ids"]]
    assert model.search([prompt], beams=1, new_tokens=len(ids))[0][0][1] == ids


@pytest.mark.gpu
def test_prompts_longer_than_a_pass_and_searches_in_a_row(native_lib, tiny):
    """A prompt over several passes equals the same prompt in one; a second search on the same cache equals the first."""
    from cudallm_b200 import beam_search
    model = beam_search.BeamSearch(tiny["bf16"], rows=4, page_size=8)
    prompt = [int(t) for t in np.random.default_rng(3).integers(0, 1000, 100)]
    a = model.search([prompt], beams=4, new_tokens=5)
    b = model.search([prompt], beams=4, new_tokens=5)
    rows, beam_search.PREFILL_ROWS = beam_search.PREFILL_ROWS, 33
    try:
        c = model.search([prompt], beams=4, new_tokens=5)
    finally:
        beam_search.PREFILL_ROWS = rows
    assert a == b
    assert [x[1] for x in a[0]] == [x[1] for x in c[0]]


@pytest.mark.gpu
def test_what_does_not_fit_is_refused(native_lib, tiny):
    from cudallm_b200.beam_search import BeamSearch
    model = BeamSearch(tiny["bf16"], rows=4, max_seq_len=32, page_size=8)
    for kw, code in ((dict(prompts=[[1] * 30], beams=2, new_tokens=3), 5), (dict(prompts=[[1]] * 3, beams=2, new_tokens=3), 5),
                     (dict(prompts=[[1, 1000]], beams=2, new_tokens=3), 1), (dict(prompts=[[]], beams=2, new_tokens=3), 1),
                     (dict(prompts=[[1]], beams=2, new_tokens=3, eos=1000), 1)):
        with pytest.raises(CudaLLMError) as e:
            model.search(**kw)
        assert e.value.code == code
    with pytest.raises(CudaLLMError) as e:
        BeamSearch(tiny["bf16"], max_seq_len=100000)
    assert e.value.code == 1
    few = BeamSearch(tiny["bf16"], rows=4, max_seq_len=32, page_size=8, n_pages=4)
    with pytest.raises(CudaLLMError, match="ran out of pages") as e:
        few.search([[1] * 20], beams=4, new_tokens=8)
    assert e.value.code == 5


def test_command_line_arguments(tmp_path):
    run = lambda *a: subprocess.run([sys.executable, "-m", "cudallm_b200.beam_search", *map(str, a)], capture_output=True, text=True, timeout=300)  # noqa: E731
    r = run("--help")
    assert r.returncode == 0 and "--beams" in r.stdout
    r = run(tmp_path / "none.cudallm")
    assert r.returncode != 0 and "no such file" in r.stderr
    (tmp_path / "x").write_bytes(b"x")
    r = run(tmp_path / "x", "--beams", 0)
    assert r.returncode != 0 and "must be >= 1" in r.stderr


def test_the_oracles_choices_are_far_enough_apart(tiny):
    """The comparison of token ids above says something: most of its cases have gaps above twice the tolerance."""
    gaps = [_plain_search(tiny["bf16"], p, 3, 7, None)[1] for p in PROMPTS]
    assert sum(g > 2 * TOL for g in gaps) >= 1, gaps


def _walk(rng, groups, beams, prompt, new, page, n_pages):
    """The forks of a search (as `BeamSearch.search` makes them) with random parents -> the most pages that one of them missed."""
    from oracle.paged64 import fork_ref
    width = -(-(prompt + new) // page)
    tables, lens, refs, worst, _ = fork_ref(np.full((groups, width), -1), np.zeros(groups, int), np.zeros(n_pages, int), range(groups), page, prompt)
    lens = np.full(groups, prompt)
    parents = np.arange(groups).repeat(beams)
    for step in range(new - 1):
        tables, lens, refs, missing, _ = fork_ref(tables, lens, refs, parents, page, 1)
        worst, lens = max(worst, missing), lens + 1
        parents = (rng.integers(0, beams, (groups, beams)) + beams * np.arange(groups)[:, None]).reshape(-1)
    return worst


@pytest.mark.parametrize("groups, beams, prompt, new, page", [(1, 4, 4, 8, 16), (1, 4, 5, 20, 16), (4, 4, 5, 20, 16), (1, 8, 8, 24, 16), (1, 4, 32, 32, 64), (2, 3, 1, 15, 4), (1, 64, 3, 9, 5),
                                                              (3, 5, 7, 30, 1)])
def test_the_pool_has_room_for_every_search_that_fits(groups, beams, prompt, new, page):
    """Pages that beams leave are free only after the step in which others take new ones: the pool holds both."""
    from cudallm_b200.beam_search import pool_pages
    for seed in range(30):
        assert _walk(np.random.default_rng(seed), groups, beams, prompt, new, page, pool_pages(groups * beams, prompt + new, page)) == 0, seed


@pytest.mark.gpu
@pytest.mark.parametrize("beams, prompt, new, page", [(4, 4, 8, 16), (8, 5, 20, 16), (3, 9, 7, 4), (4, 3, 13, 8)])
def test_searches_that_just_fit(native_lib, tiny, beams, prompt, new, page):
    """With a cache of exactly the tokens that are asked for, a search finds what it finds with room to spare."""
    from cudallm_b200.beam_search import BeamSearch
    tight, roomy = (BeamSearch(tiny["bf16"], rows=2 * beams, max_seq_len=n, page_size=page) for n in (prompt + new, 128))
    for seed in range(5):
        prompts = [[int(t) for t in np.random.default_rng([seed, g]).integers(0, 1000, prompt)] for g in range(2)]
        assert tight.search(prompts, beams=beams, new_tokens=new) == roomy.search(prompts, beams=beams, new_tokens=new)


CASES = next(m for m in test_against_a_plain_search.pytestmark if m.name == "parametrize").args[1]


@pytest.mark.parametrize("dtype, beams, page, eos", CASES)
def test_every_comparison_reaches_the_token_ids(tiny, dtype, beams, page, eos):
    """In each case of the comparison with a plain search, the token ids of one prompt or more are compared (its gap is above twice the tolerance)."""
    if eos is not None:
        eos = _plain_search(tiny[dtype], PROMPTS[0], beams, 2, None)[0][1][1][0]
    assert any(_plain_search(tiny[dtype], p, beams, 7, eos)[1] > 2 * TOL for p in PROMPTS)
