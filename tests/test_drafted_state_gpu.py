"""What a step of drafted trees leaves in a decode state, and what it takes from its arguments."""
import numpy as np
import pytest
import torch

from tests.test_drafted_gpu import DEV, SPECS, _close, _model, _prefilled
from ultraviolet_b200.drafted import TreeRunner, generate_drafted

pytestmark = pytest.mark.gpu


def _caches(st, rows=slice(None)):
    return [t[rows].clone() for y in (st.k, st.v, st.k_scale, st.v_scale) for t in y]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def _runner(m, prompts, max_new, slots=0, **kw):
    """A runner over the prompts (of one length), prefilled."""
    text = torch.tensor(prompts)
    B, n = text.shape
    st = m.new_state(B, slots or n + max_new + 2 * 64)
    if n > 1:
        m.prefill(text[:, :-1].to(DEV), torch.zeros(B, dtype=torch.long, device=DEV), st)
    return TreeRunner(m, st, text.int().to(DEV), torch.full((B,), n), max_new, **kw)


def _favour(m, *tokens):
    """Biases that make every draw one of the tokens, the first one first."""
    return dict(bias_ids=torch.tensor(tokens, dtype=torch.int32, device=DEV),
                bias=torch.tensor([1e4 - 100 * i for i in range(len(tokens))], device=DEV))


@pytest.mark.parametrize("name", sorted(SPECS))
def test_capturing_a_step_leaves_the_state_as_it_is(name):
    """Prompts longer than the window, so that an accepted path wraps over ring slots that the first step still reads, and a first draft
    that is accepted for certain: the text ends in a token that every draw is."""
    m = _model(name)
    V, n = m.cfg.vocab_size, m.cfg.window + 9
    r = np.random.default_rng(3)
    prompts = [r.integers(20, V, n - 4).tolist() + [7] * 4 for _ in range(3)]
    runs = [_runner(m, prompts, 20, branches=1, depth=5, temperature=0.0, seed=1, use_graph=g, **_favour(m, 7)) for g in (True, False)]
    graph, eager = runs
    before, pos = _caches(graph.st), graph.st.pos.clone()
    graph._capture()
    assert _same(_caches(graph.st), before) and torch.equal(graph.st.pos, pos) and int(graph.drawn.max()) == 0
    for run in runs:
        run.step()
        assert run.drawn.tolist() == [6] * 3 and torch.equal(run.st.pos, pos + 6)
    _close(graph.logits, eager.logits)
    m.engine.check_status()


def test_a_row_that_has_stopped_keeps_its_cache():
    """Row 0 stops in the first step, row 1 goes on: nothing of row 0 moves any more, whatever its ring has room for."""
    m = _model("tiny")
    V, n, eos = m.cfg.vocab_size, m.cfg.window + 9, 9
    r = np.random.default_rng(3)
    words = torch.zeros(2, (V + 31) // 32, dtype=torch.int32, device=DEV)
    words[0, 0], words[1, 0] = 1 << eos, 1 << 7
    run = _runner(m, [r.integers(20, V, n - 4).tolist() + [t] * 4 for t in (eos, 7)], 30, branches=1, depth=5, seed=1, eos_id=eos, allowed=words)
    run.step()
    assert run.done.tolist() == [True, False]
    before, pos = _caches(run.st, slice(0, 1)), run.st.pos.clone()
    for _ in range(3):
        run.step()
    assert _same(_caches(run.st, slice(0, 1)), before) and int(run.st.pos[0]) == int(pos[0]) and int(run.st.pos[1]) > int(pos[1])
    run.run()
    assert run.completions() == [[eos], [7] * 30]


@pytest.mark.parametrize("branches,depth", [(0, 1), (1, 4), (2, 3)])
@pytest.mark.parametrize("kind", ["frequency", "presence"])
def test_the_prompts_last_token_is_not_a_drawn_one(kind, branches, depth):
    """Penalties for drawn tokens leave the first draw free to repeat the prompt's last token, and no later one."""
    m = _model("tiny")
    prompts = [[3, 4, 5, 3, 4, 5, 3, 4], [7], [2, 9, 2, 9, 2]]
    for p in prompts:
        a = p[-1]
        out = generate_drafted(m, [p], 6, group=2, branches=branches, depth=depth, temperature=0.0, logit_bias={a: 500.0}, **{kind: 1000.0})
        assert all(r[0] == a and a not in r[1:] for r in out[0]), out


def test_steps_of_two_states_do_not_meet():
    """tree_step on one state, tree_step on another, then both accepts: each state takes its own nodes."""
    m = _model("tiny")
    V, T = m.cfg.vocab_size, 5
    g = torch.Generator(device=DEV).manual_seed(5)
    parents = torch.arange(-1, T - 1, device=DEV, dtype=torch.int32)
    idx = [np.random.default_rng(i).integers(1, V, (3, 6)) for i in range(2)]
    tok = [torch.randint(0, V, (3, T), generator=g, device=DEV) for _ in range(2)]
    target = [torch.cat([t[:, 1:], t[:, :1]], 1) for t in tok]                    # all of it is accepted
    new = lambda: [_prefilled(m, i, np.zeros(3, np.int64), 40) for i in idx]
    apart, mixed = new(), new()
    for st, t, y in zip(apart, tok, target):
        m.tree_step(t, parents, st)
        m.tree_accept(t, y, parents, st)
    for st, t in zip(mixed, tok):
        m.tree_step(t, parents, st)
    for st, t, y in zip(mixed, tok, target):
        m.tree_accept(t, y, parents, st)
    for a, b in zip(apart, mixed):
        assert torch.equal(a.pos, b.pos) and int(a.pos.min()) == 6 + T and _same(_caches(a), _caches(b))
    # an accept without its step, or of a step of another shape
    st = new()[0]
    with pytest.raises(RuntimeError):
        m.tree_accept(tok[0], target[0], parents, st)
    m.tree_step(tok[0], parents, st)
    with pytest.raises(RuntimeError):
        m.tree_accept(tok[0][:, :3], target[0][:, :3], parents[:3], st)


def test_tokens_of_any_layout():
    m = _model("tiny")
    V = m.cfg.vocab_size
    idx = np.random.default_rng(1).integers(1, V, (4, 6))
    st = _prefilled(m, idx, np.zeros(4, np.int64), 40)
    text = torch.randint(0, V, (4, 9), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    one, two = torch.tensor([-1], device=DEV), torch.tensor([-1, 0], device=DEV)
    for tok, parents in ((text[:, -1:], one), (text[:, 2:7:4], two), (text.t()[:2].t(), two)):
        assert torch.equal(m.tree_step(tok, parents, st), m.tree_step(tok.contiguous(), parents, st))


def test_tokens_of_any_integer_type_and_no_others():
    m = _model("tiny")
    idx = np.random.default_rng(1).integers(1, m.cfg.vocab_size, (4, 6))
    st = _prefilled(m, idx, np.zeros(4, np.int64), 40)
    tok = torch.randint(0, 100, (4, 2), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    parents = torch.tensor([-1, 0], device=DEV)
    want = m.tree_step(tok, parents, st)
    for dtype in (torch.int32, torch.int16, torch.uint8):
        assert torch.equal(m.tree_step(tok.to(dtype), parents, st), want)
    with pytest.raises(ValueError):
        m.tree_step(tok.float(), parents, st)
    with pytest.raises(ValueError):
        m.tree_step(tok.flatten(), parents, st)
    with pytest.raises(RuntimeError):
        m.tree_step(tok.cpu(), parents, st)


def test_a_tree_of_another_width_is_refused():
    """Before anything is launched: the step would read positions that the tree does not have."""
    m = _model("tiny")
    idx = np.random.default_rng(1).integers(1, m.cfg.vocab_size, (2, 6))
    st = _prefilled(m, idx, np.zeros(2, np.int64), 40)
    tok = torch.zeros((2, 4), dtype=torch.int64, device=DEV)
    for parents in ([-1], [-1, 0, 0], [-1, 0, 0, 0, 0], [[-1, 0, 0, 0]], [[-1, 0, 0]] * 2, [[-1, 0, 0, 0]] * 3):
        with pytest.raises(ValueError):
            m.tree_step(tok, torch.tensor(parents, device=DEV), st)


def test_prompt_lengths_that_the_text_does_not_have():
    m = _model("tiny")
    text = torch.ones(2, 4, dtype=torch.int32, device=DEV)
    for lens in ([0, 4], [4, 5], [-1, 2]):
        for where in ("cpu", DEV):
            with pytest.raises(ValueError):
                TreeRunner(m, m.new_state(2, 64), text, torch.tensor(lens, device=where), 8, 1, 3)


def test_allowed_tokens_outside_the_vocabulary_allow_nothing():
    m = _model("tiny")
    V = m.cfg.vocab_size
    out = generate_drafted(m, [[1, 2, 3]], 5, branches=1, depth=3, temperature=0.0, allowed_ids=[7, -1, V, V + 31, 2 ** 40],
                           logit_bias={V - 1: 1e4})
    assert out == [[[7] * 5]]


def test_the_hosts_positions_follow_a_run():
    m = _model("tiny")
    run = _runner(m, [[1, 2, 3, 4], [4, 3, 2, 1]], 12, branches=1, depth=3, temperature=0.0)
    run.run()
    assert run.st.host_pos.tolist() == run.st.pos.tolist() and int(run.st.pos.min()) >= 3 + 12


def test_a_first_step_that_is_refused_leaves_the_run_as_it_was():
    m = _model("tiny")
    run = _runner(m, [[1, 2, 3, 4], [4, 3, 2, 1]], 6, branches=1, depth=3, temperature=0.0, **_favour(m, 7))
    run.adjust["allowed"] = torch.full((2, 1), -1, dtype=torch.int32, device=DEV)      # too few words for the vocabulary
    parents = run.parents.clone()
    with pytest.raises(ValueError):
        run.step()
    assert torch.equal(run.parents, parents) and run.steps_run == 0
    run.adjust["allowed"] = None
    run.run()
    assert run.completions() == [[7] * 6] * 2
