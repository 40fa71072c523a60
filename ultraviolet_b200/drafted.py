"""Generation from drafted tokens: a prompt is prefilled once for a whole group of completions, and every step checks a tree of drafted
tokens per row instead of taking one token.

One step of ``TreeRunner``: the nodes of all trees through the layers (``DecodeEngine.tree_trunk``: kernels.tree_attention), the head,
kernels.adjust_logits, the sampler at every node, kernels.tree_advance, and the next drafts, captured in one CUDA graph.  What a row draws
behind a text is keyed by (seed, row, number of tokens drawn before), whatever tree the text stands in, so drafts decide how many
steps a completion takes and not what it says: it is what ``generate`` would give, up to the rounding of products over other batch sizes.

Drafts come from the row's own text: the continuations of the latest places where its last two tokens (else its last one) stand.
"""
from __future__ import annotations

import torch
from torch import Tensor

from .fast_decode import _engine
from .generate import _left_pad, _new_state, fresh_seed
from .kernels import adjust_logits, tree_positions


def lookup_drafts(text: Tensor, length: Tensor, branches: int, depth: int) -> tuple[Tensor, Tensor]:
    """(tokens (B, 1 + branches * depth) int64, parents int32) from text (B, n), of which row b has length[b] + 1 tokens: the last one is the
    tree's root, and behind it stand up to ``branches`` chains of ``depth`` tokens, each what follows an earlier occurrence of
    the last two tokens or, behind those, of the last one; the latest first.  An occurrence nearer than ``depth`` goes on periodically, chains
    without one are absent."""
    B, n = text.shape
    dev = text.device
    j = torch.arange(n, device=dev)
    end = length[:, None]
    last = text.gather(1, end)
    before = text.gather(1, (end - 1).clamp_min(0))
    one = (text == last) & (j < end)
    two = one & (torch.roll(text, 1, 1) == before) & (j > 0)
    at = torch.where(two, j + n, torch.where(one, j, -1)).topk(min(branches, n), 1).values       # (B, branches)
    if at.size(1) < branches:
        at = torch.cat([at, at.new_full((B, branches - at.size(1)), -1)], 1)
    real = (at >= 0)[:, :, None].expand(B, branches, depth)
    at = torch.where(at >= 0, at % n, 0)
    idx = at[:, :, None] + 1 + torch.arange(depth, device=dev) % (end - at).clamp_min(1)[:, :, None]   # (B, branches, depth)
    tokens = torch.where(real, text.gather(1, idx.clamp_max(n - 1).view(B, -1)).view_as(idx), 0).view(B, -1)
    before = torch.arange(branches * depth, device=dev, dtype=torch.int32).view(branches, depth).clone()
    before[:, 0] = 0                                                                              # node i stands behind node i - 1 or the root
    parents = torch.where(real, before, -2).reshape(B, -1)
    root = torch.full((B, 1), -1, dtype=torch.int32, device=dev)
    return torch.cat([last, tokens], 1).long(), torch.cat([root, parents.to(torch.int32)], 1)


class TreeRunner:
    """Steps of drafted trees over a decode state whose rows hold all of their prompt but its last token.

    text (B, n) holds the prompts (prompt_lengths[b] >= 1 tokens from column 0) and receives what is drawn; branches chains of depth
    drafted tokens per row and step (at most 63 tokens).  repetition, frequency, presence, bias_ids / bias and allowed are those of
    kernels.adjust_logits.  A row stops at eos_id or after max_new tokens; ``completions`` returns what was drawn."""

    def __init__(self, model, st, text: Tensor, prompt_lengths: Tensor, max_new: int, branches: int = 1, depth: int = 7,
                 temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, seed: int | None = None, eos_id: int | None = None,
                 repetition=None, frequency=None, presence=None, bias_ids=None, bias=None, allowed=None, use_graph: bool = True):
        self.eng, self.st = _engine(model), st
        eng, dev, B = self.eng, st.pos.device, st.B
        self.branches, self.depth, self.T = int(branches), int(depth), 1 + int(branches) * int(depth)
        if self.branches < 0 or self.depth < 1 or self.T > 64:
            raise ValueError("a tree has at most 64 nodes: the last token and branches * depth drafted ones")
        if text.shape[0] != B or prompt_lengths.shape != (B,):
            raise ValueError(f"one text and one prompt length for each of {B} rows")
        if B and not (1 <= int(prompt_lengths.min()) and int(prompt_lengths.max()) <= text.size(1)):   # (they index the text)
            raise ValueError(f"prompts have 1 to {text.size(1)} tokens, as the text does")
        # (a row's last tree may end T tokens behind the last one wanted; the other T are room for one more tree behind it)
        if st.max_len < text.size(1) + int(max_new) + 2 * self.T:
            raise ValueError(f"the state has {st.max_len} slots a row; {text.size(1)} + {max_new} tokens in trees of {self.T} need "
                             f"{text.size(1) + int(max_new) + 2 * self.T}")
        self.temperature, self.top_k, self.top_p = temperature, int(top_k or 0), top_p
        self.seed = fresh_seed() if seed is None else int(seed)
        self.max_new, self.eos_id, self.use_graph = int(max_new), eos_id, use_graph
        # the texts, with a column behind them for what is written nowhere; rows of a multiple of 16 bytes
        self.cap = (text.size(1) + self.max_new + self.T + 3) // 4 * 4
        self.text = torch.zeros(B, self.cap + 4, dtype=torch.int32, device=dev)
        self.text[:, :text.size(1)] = text
        self.prompt = prompt_lengths.to(device=dev, dtype=torch.int64).contiguous()
        self.length = self.prompt - 1                      # tokens in front of the root
        self.drawn = torch.zeros(B, dtype=torch.int64, device=dev)
        self.done = torch.zeros(B, dtype=torch.bool, device=dev)
        self.tok, self.parents = self._drafts()
        M, V = B * self.T, eng.cfg.vocab_size
        row = lambda v: None if v is None else v if isinstance(v, Tensor) else torch.full((B,), float(v), dtype=torch.float32, device=dev)
        self.adjust = dict(repetition=row(repetition), frequency=row(frequency), presence=row(presence), bias_ids=bias_ids, bias=bias,
                           allowed=allowed)
        self.head = torch.empty(M, V, dtype=eng.dtype, device=dev)
        self.logits = torch.empty(B, self.T, V, dtype=torch.float32, device=dev)
        self.target = torch.zeros(M, dtype=torch.int64, device=dev)
        self.logp = torch.zeros(M, dtype=torch.float32, device=dev)
        self.row_keys = torch.arange(B, dtype=torch.int64, device=dev).repeat_interleave(self.T)
        self.steps_run, self.graph = 0, None

    def _drafts(self):
        if self.branches == 0:
            tok = self.text.gather(1, self.length[:, None]).long()
            parents = torch.full((tok.size(0), 1), -1, dtype=torch.int32, device=tok.device)
        else:
            tok, parents = lookup_drafts(self.text[:, :self.cap], self.length, self.branches, self.depth)
        # a row that has stopped gets a tree without nodes: it draws nothing, and nothing of it moves
        return tok, torch.where(self.done[:, None], -2, parents)

    def _body(self) -> None:
        st, eng, T = self.st, self.eng, self.T
        B = st.B
        h = eng.tree_trunk(self.tok, self.parents, st)
        torch.mm(h, eng.w["embed"].t(), out=self.head)
        # the root stands in the text, where it counts as what it is: in the first step as the prompt's last token, then as a drawn one
        drafted = self.tok.clone()
        drafted[:, 0] = -1
        adjust_logits(self.head.view(B, T, -1), softcap=eng.cfg.softcap, history=self.text, lengths=self.length + 1,
                      prompt_lengths=self.prompt, parents=self.parents, tokens=drafted, out=self.logits, **self.adjust)
        steps = tree_positions(self.parents, self.drawn).view(-1)
        eng.sample(self.logits.view(B * T, -1), self.temperature, self.top_p, seed=self.seed, row_keys=self.row_keys, steps=steps,
                   tok_out=self.target, logp_out=self.logp, precapped=True, top_k=self.top_k)
        _, count, new = eng.tree_advance(self.tok, self.target.view(B, T), self.parents, st)
        j = torch.arange(T, device=new.device)
        live = j < count[:, None]
        self.text.scatter_(1, torch.where(live, self.length[:, None] + 1 + j, self.cap), new.to(torch.int32))
        self.length += count
        self.drawn += count
        self.done |= self.drawn >= self.max_new
        if self.eos_id is not None:
            self.done |= ((new == self.eos_id) & live).any(1)
        tok, parents = self._drafts()
        self.tok.copy_(tok)
        self.parents.copy_(parents)

    def step(self) -> None:
        """One step of every row that has not stopped."""
        if not self.use_graph:
            self._body()
        else:
            if self.graph is None:
                self._capture()
            self.graph.replay()
        self.steps_run += 1

    def _capture(self) -> None:
        dev = self.st.pos.device
        kept = [self.st.pos, self.text, self.length, self.drawn, self.done, self.tok, self.parents]
        saved = [t.clone() for t in kept]
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        try:
            with torch.cuda.stream(s):
                # warm-up without a node in any tree: an accepted path would wrap over ring slots that the real first step still reads
                self.parents.fill_(-2)
                self._body()
        finally:
            torch.cuda.current_stream(dev).wait_stream(s)
            for t, v in zip(kept, saved):
                t.copy_(v)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            self._body()
        self.graph = g

    def run(self, check_every: int = 8) -> None:
        """Steps until every row has stopped."""
        while not bool(self.done.all()):
            for _ in range(check_every):
                self.step()
        self.st.host_pos[:] = self.st.pos.cpu().numpy()         # (what goes on with the state plans by it)
        self.eng.check_status(self.st.B * self.T)

    def completions(self) -> list[list[int]]:
        text, first, n = self.text.tolist(), self.prompt.tolist(), self.drawn.tolist()
        rows = [t[a:a + min(k, self.max_new)] for t, a, k in zip(text, first, n)]
        return [r if self.eos_id is None or self.eos_id not in r else r[:r.index(self.eos_id) + 1] for r in rows]


@torch.no_grad()
def generate_drafted(model, prompts, max_new: int, group: int = 1, branches: int = 1, depth: int = 7, temperature: float = 1.0,
                     top_k: int = 0, top_p: float = 1.0, eos_id: int | None = None, pad_id: int = 0, seed: int | None = None,
                     repetition: float | None = None, frequency: float | None = None, presence: float | None = None,
                     logit_bias: dict[int, float] | None = None, allowed_ids=None, use_graph: bool = True, stats: dict | None = None):
    """``group`` completions of every prompt, a list of lists per prompt.  The prompts are prefilled once and their cache rows forked to their
    groups; every step then checks ``branches`` drafted chains of ``depth`` tokens per row (branches=0: one token per step).

    repetition, frequency, presence: penalties for tokens of a row's text; logit_bias: token -> added to its logit; allowed_ids: the only
    tokens that may be drawn (kernels.adjust_logits has the formulas).  seed as in ``generate``: row i of prompt-major order draws from
    (seed, i).  stats: receives steps and drawn (tokens)."""
    eng = _engine(model)
    dev, n, V = eng.device, len(prompts), eng.cfg.vocab_size
    if group < 1 or any(len(p) == 0 for p in prompts):
        raise ValueError("generate_drafted takes groups of at least one row and prompts of at least one token")
    B, T = n * group, 1 + branches * depth
    if B == 0 or max_new < 1:
        return [[[] for _ in range(group)] for _ in range(n)]
    idx, starts = _left_pad(prompts, pad_id, dev)
    st = _new_state(model, B, idx.size(1) + max_new + 2 * T, eng, 0)
    lead = torch.arange(0, B, group, device=dev)
    if idx.size(1) > 1:
        model.prefill(idx[:, :-1], starts, st, rows=lead)
    else:
        st.starts[lead] = starts
    st.fork([i - i % group for i in range(B) if i % group], [i for i in range(B) if i % group])
    lens = torch.tensor([len(p) for p in prompts])
    text = torch.zeros(n, int(lens.max()), dtype=torch.int32)
    for i, p in enumerate(prompts):
        text[i, :len(p)] = torch.as_tensor(p, dtype=torch.int32)
    bias_ids = bias = allowed = None
    if logit_bias:
        bias_ids = torch.tensor(list(logit_bias), dtype=torch.int32, device=dev)
        bias = torch.tensor([float(v) for v in logit_bias.values()], dtype=torch.float32, device=dev)
    if allowed_ids is not None:
        bits = torch.zeros((V + 31) // 32 * 32, dtype=torch.int64)
        ids = torch.as_tensor(list(allowed_ids), dtype=torch.int64)
        bits[ids[(ids >= 0) & (ids < V)]] = 1                   # (others are no tokens: ignored, as adjust_logits does)
        words = (bits.view(-1, 32) << torch.arange(32)).sum(1)
        allowed = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).to(dev).expand(B, -1)
    runner = TreeRunner(model, st, text.repeat_interleave(group, 0).to(dev), lens.repeat_interleave(group), max_new, branches, depth,
                        temperature, top_k, top_p, seed, eos_id, repetition, frequency, presence, bias_ids, bias, allowed, use_graph)
    runner.run()
    out = runner.completions()
    if stats is not None:
        stats.update(steps=runner.steps_run, drawn=sum(map(len, out)), slots=B)
    return [out[i * group:(i + 1) * group] for i in range(n)]
