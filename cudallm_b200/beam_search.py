"""Beam search of a .cudallm model over a paged key-value cache.

    python -m cudallm_b200.beam_search MODEL.cudallm --beams 4 --new 32 --prompt-len 64 --prompts 2

The reference decodes one sequence greedily; this runs the same per-token sequence (wasiqnauman/cudallm
src/engine/engine.cpp:181-237) for several prompts and several beams of each. The beams of a prompt share its pages;
`PagedCache.append` rotates and stores, `attend` reads, `beam_select` picks who goes on with which token and
`fork` hands the pages on. Prompts are fed through the same calls, every token of a prompt as a row of its own that sees
the tokens up to itself. The weights are expanded to fp32 on the GPU and multiplied by torch, so results compare with the
reference's fp32 model; nothing in the loop over tokens waits for the GPU.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import numpy as np
import torch

from . import format as fmt
from .abi import CudaLLMError
from .paged import PagedCache, Rope, beam_select
from .quantize import dequantize_int4_groups, dequantize_int8_rows

KV_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
PREFILL_ROWS = 512  # prompt tokens of one pass


def pool_pages(rows: int, max_seq_len: int, page_size: int) -> int:
    """Pages with which any search of `rows` sequences of up to `max_seq_len` tokens succeeds: all that the rows can hold, and one more a
    row, since a step's new pages are found before those of the beams that end in it are free."""
    return rows * (-(-max_seq_len // page_size) + 1)


class BeamSearch:
    """Beam search with a model's weights and a pool of pages for up to `rows` sequences (prompts * beams) of up to
    `max_seq_len` tokens (0: the file header's value); n_pages 0: as many as any search of that size can need."""

    def __init__(self, path: Path | str, *, rows: int = 16, max_seq_len: int = 0, page_size: int = 16, n_pages: int = 0,
                 kv_dtype: str = "fp16", device: str = "cuda"):
        self.device = torch.device(device, torch.cuda.current_device()) if device == "cuda" else torch.device(device)
        hdr = fmt.read_header(path)
        self.hidden, self.inter, self.n_layers = hdr["hidden_size"], hdr["intermediate_size"], hdr["n_layers"]
        self.heads, self.kv_heads, self.head_dim = hdr["n_heads"], hdr["n_kv_heads"], hdr["head_dim"]
        self.vocab, self.eps = hdr["vocab_size"], hdr["rms_eps"]
        if max_seq_len < 0 or max_seq_len > hdr["max_seq_len"]:
            raise CudaLLMError(1, f"max_seq_len must be in 0 .. {hdr['max_seq_len']}")
        self.max_seq_len = max_seq_len or hdr["max_seq_len"]
        table = {e["name"]: e for e in fmt.read_table(path)}

        def vector(name: str) -> torch.Tensor:
            return torch.from_numpy(fmt.load_tensor(path, table[name]).astype(np.float32)).to(self.device)

        def matrix(name: str) -> torch.Tensor:
            w = table[name + ".weight"]
            raw = fmt.load_tensor(path, w)
            if w["dtype"] == fmt.BF16:
                return torch.from_numpy(raw.view(np.int16)).to(self.device).view(torch.bfloat16).float()
            scales = fmt.load_tensor(path, table[name + ".scales"])
            if w["dtype"] == fmt.I8:
                dense = dequantize_int8_rows(raw, scales.reshape(-1))
            else:
                dense = dequantize_int4_groups(raw, scales)
            return torch.from_numpy(np.ascontiguousarray(dense, dtype=np.float32)).to(self.device)

        self.embedding, self.final_norm = matrix("tok_embeddings"), vector("norm.weight")
        self.layers = [{"attn_norm": vector(p + "attn_norm.weight"), "wqkv": matrix(p + "wqkv"), "wo": matrix(p + "wo"),
                        "ffn_norm": vector(p + "ffn_norm.weight"), "w_gate_up": matrix(p + "w_gate_up"), "w_down": matrix(p + "w_down")}
                       for p in (f"layers.{i}." for i in range(self.n_layers))]
        self.rope = Rope(vector("rope.inv_freq"))
        self.rows, self.width = rows, -(-self.max_seq_len // page_size)
        self.cache = PagedCache.allocate(self.n_layers, n_pages or pool_pages(rows, self.max_seq_len, page_size), self.kv_heads, page_size,
                                         self.head_dim, dtype=KV_DTYPES[kv_dtype], device=self.device)

    def _norm(self, x: torch.Tensor, gain: torch.Tensor) -> torch.Tensor:
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + self.eps) * gain

    def _forward(self, tokens: torch.Tensor, positions: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor) -> torch.Tensor:
        """Residual stream [rows][hidden] after the layers of one token per row, stored at `positions`, seeing `lens` tokens."""
        n = tokens.numel()
        x = self.embedding[tokens.long()]
        for i, w in enumerate(self.layers):
            qkv = (self._norm(x, w["attn_norm"]) @ w["wqkv"].T).view(n, self.heads + 2 * self.kv_heads, self.head_dim)
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
            q = self.cache.append(q, k, v, positions, tables, self.rope, layer=i, out=q)
            x = x + self.cache.attend(q, tables, lens, layer=i).view(n, -1) @ w["wo"].T
            gate, up = (self._norm(x, w["ffn_norm"]) @ w["w_gate_up"].T).split(self.inter, 1)
            x = x + (gate / (1.0 + torch.exp(-gate)) * up) @ w["w_down"].T
        return x

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        return self._norm(x, self.final_norm) @ self.embedding.T

    def _ints(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    @torch.no_grad()
    def search(self, prompts: list[list[int]], *, beams: int, new_tokens: int, eos: int | None = None) -> list[list[tuple[float, list[int]]]]:
        """For each prompt its `beams` best continuations of `new_tokens` tokens, best first, as (sum of the tokens'
        log-probabilities, token ids); one that reached `eos` stays as it is and ends there."""
        groups, rows = len(prompts), len(prompts) * beams
        lengths = [len(p) for p in prompts]
        if groups == 0 or min(lengths) == 0 or beams < 1 or new_tokens < 1:
            raise CudaLLMError(1, "search needs prompts of one token or more, one beam or more and one new token or more")
        if rows > self.rows or max(lengths) + new_tokens > self.max_seq_len:
            raise CudaLLMError(5, f"{rows} sequences of {max(lengths) + new_tokens} tokens: the cache has room for {self.rows} of {self.max_seq_len}")
        if any(not 0 <= t < self.vocab for p in prompts for t in p) or (eos is not None and not 0 <= eos < self.vocab):
            raise CudaLLMError(1, "token out of range")
        cache = self.cache
        state = cache.fork(*cache.rows(groups, self.width), self._ints(range(groups)), room=max(lengths))
        short = state[3]
        last = torch.empty((groups, self.hidden), dtype=torch.float32, device=self.device)
        for g, prompt in enumerate(prompts):
            for first in range(0, len(prompt), PREFILL_ROWS):
                part = prompt[first:first + PREFILL_ROWS]
                positions = torch.arange(first, first + len(part), dtype=torch.int32, device=self.device)
                tables = state[0][g:g + 1].repeat(len(part), 1)  # every token a row that sees the ones up to itself
                x = self._forward(self._ints(part), positions, tables, positions + 1)
            last[g] = x[-1]
        scores, parents, tokens = beam_select(self._logits(last), torch.zeros((groups, 1), device=self.device), keep=beams)
        lens = self._ints(lengths)
        ids = torch.zeros((groups, new_tokens), dtype=torch.int32, device=self.device)
        done = torch.zeros(groups, dtype=torch.int32, device=self.device)
        for n in range(new_tokens):
            who, what = parents.view(-1).long(), tokens.view(-1)
            ids = ids[who]
            ids[:, n] = what
            done = done[who] if eos is None else done[who] | (what == eos).int()
            if n + 1 == new_tokens:
                break
            state = cache.fork(state[0], lens, state[2], parents.view(-1), room=1)
            short = torch.maximum(short, state[3])
            tables, lens = state[0], state[1]
            x = self._forward(what, lens, tables, lens + 1)
            lens = lens + 1
            scores, parents, tokens = beam_select(self._logits(x), scores, keep=beams, finished=done.view(groups, beams),
                                                  eos=0 if eos is None else eos)
        if int(short) > 0:
            raise CudaLLMError(5, f"the cache ran out of pages ({int(short)} too few in one step); results are invalid")
        out = []
        for g in range(groups):
            found = []
            for b in range(beams):
                t = ids[g * beams + b].tolist()
                found.append((float(scores[g, b]), t[:t.index(eos) + 1] if eos is not None and eos in t else t))
            out.append(found)
        return out


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("model", help=".cudallm file")
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--new", type=int, default=32, help="tokens to add to each prompt")
    ap.add_argument("--prompts", type=int, default=1, help="number of seeded random prompts")
    ap.add_argument("--prompt-len", type=int, default=32)
    ap.add_argument("--prompt", type=int, nargs="+", default=None, help="token ids of one prompt, instead of random ones")
    ap.add_argument("--eos", type=int, default=None)
    ap.add_argument("--kv", choices=tuple(KV_DTYPES), default="fp16")
    ap.add_argument("--page", type=int, default=16, help="tokens of a page")
    args = ap.parse_args(argv)
    if min(args.beams, args.new, args.prompts, args.prompt_len, args.page) < 1:
        ap.error("--beams, --new, --prompts, --prompt-len and --page must be >= 1")
    if not Path(args.model).is_file():
        ap.error(f"no such file: {args.model}")
    vocab = fmt.read_header(args.model)["vocab_size"]
    prompts = [args.prompt] if args.prompt else [[int(t) for t in np.random.default_rng([0, i]).integers(0, vocab, args.prompt_len)]
                                                 for i in range(args.prompts)]
    longest = max(map(len, prompts)) + args.new
    model = BeamSearch(args.model, rows=len(prompts) * args.beams, max_seq_len=longest, page_size=args.page, kv_dtype=args.kv)
    model.search(prompts, beams=args.beams, new_tokens=min(2, args.new), eos=args.eos)  # first use of every kernel
    torch.cuda.synchronize()
    began = time.perf_counter()
    found = model.search(prompts, beams=args.beams, new_tokens=args.new, eos=args.eos)
    took = time.perf_counter() - began
    for g, beams in enumerate(found):
        for score, ids in beams:
            print(f"prompt {g}: {score:9.4f}  {' '.join(map(str, ids))}")
    print(f"{len(prompts)} prompts x {args.beams} beams x {args.new} tokens in {took:.3f} s")
    return 0


if __name__ == "__main__":
    sys.exit(main())
