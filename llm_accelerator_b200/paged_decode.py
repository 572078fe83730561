"""The model's layers in 16 bits over a paged cache: the operators of ``paged`` as
a serving loop uses them.

The fixed-point path is the product's arithmetic; ``fp32_diag`` judges it against
a float32 forward of the same weights, one position at a time.  ``PagedDecoder`` is
that float model at serving speed: prompts enter in chunks, sequences of
different lengths step together, prompts are shared by forking (and their keys read once
for neighbouring forks), texts may grow past a window whose first tokens stay visible,
tokens are judged by their log probabilities, and the cache is packed when sequences
end.  Per layer (H/common.py:231-298 in the reference):

    residual add + norm            paged.AddRmsNorm
    q, k, v product                torch.matmul (cuBLAS)
    q/k norm, rotary, K/V store    paged.RopeAppend
    attention over the pages       paged.Attention, or paged.SharedAttention for forks
    o product, residual + norm     torch.matmul, paged.AddRmsNorm
    gate/up, SiLU, down products   torch.matmul; with ``eight_bit`` the gate/up input is
                                   normed straight into e4m3 with a scale per row and
                                   multiplied in 8 bits

and of the logits                  paged.TokenLogprobs

    python -m llm_accelerator_b200.paged_decode [prompt tokens] [continuations]
"""
from __future__ import annotations

import json
import sys
from typing import Optional, Sequence

import torch

from . import _native, tables
from .fp32_diag import EPS, HEAD_DIM, HEADS, INTER, KV_HEADS, THETA
from .paged import AddRmsNorm, Attention, PagedCache, RopeAppend, SharedAttention, Step, TokenLogprobs, TokenScores


class PagedDecoder:
    """A Qwen3 layer stack with its paged cache.

    ``weights``: the dict of ``fp32_diag.float_weights``.  ``rope_factor`` above 1 stretches
    the rotary frequencies over ``max_ctx`` (``tables.rope_float_tables``).  With ``window`` a
    token sees the last ``window`` ones up to itself, and the first ``sinks``.
    """

    def __init__(self, weights: dict, max_seqs: int = 8, max_ctx: int = 4096, n_pages: Optional[int] = None,
                 page_tokens: int = 64, dtype: torch.dtype = torch.bfloat16, rope_factor: float = 1.0,
                 eight_bit: bool = False, window: int = 0, sinks: int = 0):
        T, dev = _native, weights["embed"].device
        layers = weights["layers"]
        self.dtype, self.eight_bit, self.window = dtype, eight_bit, window
        self._logprobs: dict[int, TokenLogprobs] = {}
        self.embed = weights["embed"].to(dtype)
        per_seq = -(-max_ctx // page_tokens)
        self.cache = PagedCache(len(layers), n_pages or max_seqs * per_seq, page_tokens, KV_HEADS, HEAD_DIM, max_seqs,
                                max_ctx, dtype, dev)
        cos, sin = tables.rope_float_tables(max_ctx, HEAD_DIM, THETA, rope_factor, device=dev)
        self.final = AddRmsNorm(weights["final"].to(dtype), EPS)
        self.layers = []
        for i, w in enumerate(layers):
            def cat(*ids):
                return torch.cat([w[t] for t in ids]).to(dtype)
            k, v = self.cache.k(i), self.cache.v(i)
            lay = {"qkv": cat(T.T_Q, T.T_K, T.T_V), "o": cat(T.T_O), "gu": cat(T.T_GATE, T.T_UP), "down": cat(T.T_DOWN),
                   "norm1": AddRmsNorm(w[T.T_INPUT_GAMMA].to(dtype), EPS),
                   "norm2": AddRmsNorm(w[T.T_POST_GAMMA].to(dtype), EPS,
                                       out_dtype=torch.float8_e4m3fn if eight_bit else None),
                   "rope": RopeAppend(cos, sin, q_gamma=w[T.T_Q_GAMMA].to(dtype), k_gamma=w[T.T_K_GAMMA].to(dtype),
                                      eps=EPS),
                   "attn": Attention(k, v, self.cache.table, self.cache.lens, q_heads=HEADS, window=window, sinks=sinks),
                   "k": k, "v": v}
            if eight_bit:
                top = lay["gu"].float().abs().amax(1, keepdim=True) / 448.0
                top[top == 0] = 1.0  # a row of zeros stays zeros
                lay["gu8"] = (lay["gu"].float() / top).to(torch.float8_e4m3fn)
                lay["gu8_scale"] = top.t().contiguous()
            self.layers.append(lay)

    def _attend(self, lay: dict, q: torch.Tensor, step: Step) -> torch.Tensor:
        if step.cu_group is None or self.window:
            return lay["attn"](q, None, step.cu_q, max_q=step.max_q, max_ctx=step.max_ctx, seq_ids=step.seq_ids)
        if "shared" not in lay:
            lay["shared"] = SharedAttention(lay["k"], lay["v"], self.cache.table, self.cache.lens, q_heads=HEADS,
                                            share=self.layers[0].get("shared"))  # the layers run one after another
        return lay["shared"](q, None, step.cu_q, step.cu_group, step.prefix_lens, max_q=step.max_q,
                             max_ctx=step.max_ctx, max_prefix=step.max_prefix, seq_ids=step.seq_ids)

    def _known(self, tokens: Sequence[Sequence[int]]) -> None:
        vocab = self.embed.shape[0]
        if not all(0 <= t < vocab for one in tokens for t in one):
            raise ValueError(f"a token is outside the vocabulary of {vocab}")

    def _layers(self, seqs: Sequence[int], tokens: Sequence[Sequence[int]]) -> tuple[torch.Tensor, torch.Tensor, Step]:
        """Appends tokens[i] to sequence seqs[i]; the last layer's residual stream and what is still to be added to it."""
        counts = [len(t) for t in tokens]
        if min(counts, default=0) < 1:
            raise ValueError("every sequence of a step needs a token")
        self._known(tokens)
        flat = torch.tensor([t for one in tokens for t in one], dtype=torch.long).pin_memory()
        step = self.cache.extend(seqs, counts)
        h = self.embed[flat.to(self.embed.device, non_blocking=True)]
        n = h.shape[0]
        add = None
        for lay in self.layers:
            # h becomes h + add, the layer's input; x is its norm
            x = lay["norm1"](h if add is None else add, residual=None if add is None else h,
                             residual_out=None if add is None else h)
            qkv = (x @ lay["qkv"].t()).view(n, HEADS + 2 * KV_HEADS, HEAD_DIM)
            q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]
            lay["rope"](q, k, v, step.positions, step.rows, lay["k"], lay["v"])
            add = self._attend(lay, q, step).view(n, HEADS * HEAD_DIM) @ lay["o"].t()
            if self.eight_bit:
                x8, s8 = lay["norm2"](add, residual=h, residual_out=h)
                gu = torch._scaled_mm(x8, lay["gu8"].t(), scale_a=s8, scale_b=lay["gu8_scale"], out_dtype=self.dtype)
            else:
                gu = lay["norm2"](add, residual=h, residual_out=h) @ lay["gu"].t()
            add = (torch.nn.functional.silu(gu[:, :INTER]) * gu[:, INTER:]) @ lay["down"].t()
        return h, add, step

    def forward(self, seqs: Sequence[int], tokens: Sequence[Sequence[int]]) -> torch.Tensor:
        """Appends tokens[i] to sequence seqs[i]; float32 logits [sequences, vocab] after each one's last token."""
        h, add, step = self._layers(seqs, tokens)
        last = step.cu_q[1:].long() - 1
        return (self.final(add[last], residual=h[last]) @ self.embed.t()).float()

    def logprobs(self, top: int = 0) -> TokenLogprobs:
        """The decoder's ``TokenLogprobs`` with ``top`` alternatives."""
        if top not in self._logprobs:
            self._logprobs[top] = TokenLogprobs(top, self.embed.device)
        return self._logprobs[top]

    def score(self, seq: int, tokens: Sequence[int], chunk: int = 512, top: int = 0) -> list[TokenScores]:
        """Appends `tokens` to a sequence in chunks and judges each by the one before it: row i of a chunk is about the
        token that follows its token i (the last row of all about none: logprob 0, rank 0)."""
        if not len(tokens) or chunk < 1:
            raise ValueError("a text has a token and a chunk at least one")
        self._known([tokens])
        judge, scores = self.logprobs(top), []
        targets = torch.tensor(list(tokens[1:]) + [-1], dtype=torch.long).to(self.embed.device)
        for at in range(0, len(tokens), chunk):
            h, add, _ = self._layers([seq], [tokens[at:at + chunk]])
            scores.append(judge(self.final(add, residual=h) @ self.embed.t(), targets[at:at + chunk]))
        return scores

    def prefill(self, seq: int, prompt: Sequence[int], chunk: int = 512) -> torch.Tensor:
        """A prompt in chunks; the logits after its last token."""
        if not len(prompt) or chunk < 1:
            raise ValueError("a prompt has a token and a chunk at least one")
        for at in range(0, len(prompt), chunk):
            logits = self.forward([seq], [prompt[at:at + chunk]])
        return logits

    def generate(self, seqs: Sequence[int], logits: torch.Tensor, n: int) -> list[list[int]]:
        """n greedy tokens of every sequence, from the logits after its last one."""
        return self._greedy(seqs, logits, n, lambda x: (x.argmax(-1).tolist(), None))[0]

    def generate_scored(self, seqs: Sequence[int], logits: torch.Tensor, n: int) -> \
            tuple[list[list[int]], list[list[float]]]:
        """n greedy tokens of every sequence and their log probabilities."""
        judge = self.logprobs(1)

        def pick(x: torch.Tensor) -> tuple[list[int], list[float]]:
            best = judge(x)
            return best.top_index[:, 0].tolist(), best.top_logprob[:, 0].tolist()
        return self._greedy(seqs, logits.to(self.embed.device), n, pick)

    def _greedy(self, seqs: Sequence[int], logits: torch.Tensor, n: int, pick) -> \
            tuple[list[list[int]], list[list[float]]]:
        """n tokens of every sequence by `pick`, which gives those of one step's logits, and their scores or None."""
        out, scores = [[] for _ in seqs], [[] for _ in seqs]
        for i in range(n):
            tokens, values = pick(logits)
            for o, t in zip(out, tokens):
                o.append(t)
            for s, v in zip(scores, values or ()):
                s.append(v)
            if i + 1 < n:
                logits = self.forward(seqs, [[t] for t in tokens])
        return out, scores


def run(prompt_tokens: int = 1500, continuations: int = 4, new_tokens: int = 8, n_layers: int = 4, vocab: int = 4096,
        seed: int = 0, chunk: int = 512) -> dict:
    """One prompt shared by several continuations on the synthetic model: prefilled in chunks,
    forked, continued by different first tokens together, ended but one, packed, continued; with the mean log
    probability of each continuation's tokens."""
    from .fp32_diag import float_weights

    class Shape:  # what float_weights asks of a model
        pass

    Shape.vocab, Shape.n_layers = vocab, n_layers
    d = PagedDecoder(float_weights(Shape, seed), max_seqs=continuations + 1, max_ctx=prompt_tokens + 4 * new_tokens + 2)
    g = torch.Generator().manual_seed(seed)
    prompt = torch.randint(0, vocab, (prompt_tokens,), generator=g).tolist()
    logits = d.prefill(0, prompt, chunk)
    kids = list(range(1, continuations + 1))
    d.cache.fork(0, kids)
    starts = logits[0].topk(continuations).indices.tolist()
    texts, scores = d.generate_scored(kids, d.forward(kids, [[t] for t in starts]), new_tokens)
    used = d.cache.pool.shape[0] - d.cache.free_pages
    for s in [0] + kids[:-1]:
        d.cache.free(s)
    live = d.cache.compact()
    more = d.generate(kids[-1:], d.forward(kids[-1:], [[texts[-1][-1]]]), new_tokens)
    d.cache.pages.check()
    return {"prompt_tokens": prompt_tokens, "continuations": {t: x for t, x in zip(starts, texts)},
            "logprobs": {t: sum(s) / len(s) for t, s in zip(starts, scores)}, "pages_used": used,
            "pages_after_compaction": live, "continued": more[0]}


if __name__ == "__main__":
    print(json.dumps(run(*(int(x) for x in sys.argv[1:3]))))
