"""Values and layouts at which the tree kernels have to agree with their formulas and with each other."""
import pytest
import torch

from oracle import tree as ot
from tests.test_tree_gpu import UNIT, _gen, _np, _state, _tree

pytestmark = pytest.mark.gpu

# one call for each way through the kernels: B, T, H, K, hd, S, num_splits
ROUTES = {
    "rows, whole": (3, 3, 8, 1, 64, 90, 1),
    "rows, parts in a cluster": (3, 6, 8, 1, 64, 700, 4),
    "rows, parts in the workspace": (3, 5, 8, 2, 128, 2000, 12),
    "rows, plain copies": (3, 4, 4, 2, 32, 91, 1),
    "128 rows a unit, whole": (90, 16, 8, 1, 64, 130, None),
    "128 rows a unit, cut": (3, 40, 8, 1, 64, 60000, None),
    "two tiles at a time, whole": (256, 8, 8, 1, 64, 500, None),
    "two tiles at a time, cut": (16, 5, 8, 1, 64, 70000, None),
    "head_dim 128, cut": (4, 40, 8, 2, 128, 30000, None),
}


def _call(route, dtype=torch.bfloat16, kind="random"):
    from ultraviolet_b200.kernels import tree_attention
    B, T, H, K, hd, S, splits = ROUTES[route]
    kc, vc, ks, vs = _state(B, K, S, hd, dtype, T)
    x = torch.randn((B, T, H + 2 * K, hd), generator=_gen(T), device="cuda").to(dtype)
    pos = torch.arange(B, device="cuda") * 7 % 30 + (S - 30)
    par = torch.tensor(_tree(kind, B, T, T), device="cuda")

    def run(x, ks=ks, vs=vs, **kw):
        return tree_attention(x[:, :, :H], x[:, :, H:H + K], x[:, :, H + K:], kc, vc, pos, pos * 0, par, 0.14, k_scale=ks, v_scale=vs,
                              num_splits=splits, **kw)
    return run, x, ks, vs, pos, par


@pytest.mark.parametrize("route", sorted(ROUTES))
def test_what_is_not_finite_shows(route):
    """A present node whose query, or a visible key's scale, is no number has no softmax: NaN on every route, and nothing else changes."""
    B, T, H, K, hd, S, splits = ROUTES[route]
    run, x, ks, vs, pos, par = _call(route)
    want = run(x)
    y = x.clone()
    hit = [(0, T - 1, 1, float("nan")), (1, 0, 0, float("inf")), (2, 1, H - 1, float("-inf"))]
    for b, t, h, v in hit:
        y[b, t, h, 3] = v
    y[0, 1, 2] = float("nan")
    hit.append((0, 1, 2, None))
    got, keep = run(y), torch.ones_like(want[..., 0], dtype=torch.bool)
    for b, t, h, _ in hit:
        assert got[b, t, h].isnan().all(), (b, t, h)
        keep[b, t, h] = False
    assert torch.equal(got[keep], want[keep])
    # a visible key's scale: all nodes of that row, and of the kv head's query heads
    bad = ks.clone()
    bad[1, K - 1, S // 2] = float("nan")
    got, keep = run(x, ks=bad), torch.ones_like(want[..., 0], dtype=torch.bool)
    keep[1, :, H - H // K:] = False
    assert got[~keep].isnan().all() and torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("route", sorted(ROUTES))
def test_absent_nodes_get_zeros_whatever_they_hold(route):
    run, x, ks, vs, pos, par = _call(route, kind="padded")
    par[:, 1] = -2
    y = x.clone()
    y[:, 1] = float("nan")
    want, got = run(x), run(y)
    assert (got[:, 1] == 0).all() and torch.equal(got, want)


def test_watched_calls_count_what_they_skip():
    from torch.utils._python_dispatch import TorchDispatchMode
    from ultraviolet_b200.kernels import kv_fork, tree_advance

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    B, T, S = 3, 4, 20
    kc, vc, ks, vs = _state(B, 1, S, 64, torch.bfloat16, 1)
    x = torch.randn((B, T, 2, 64), generator=_gen(1), device="cuda").to(torch.bfloat16)
    par, tok = torch.arange(-1, T - 1, device="cuda"), torch.zeros((B, T), dtype=torch.long, device="cuda")
    new = lambda: torch.zeros(1, dtype=torch.int32, device="cuda")
    dev = lambda *a: torch.tensor(a, device="cuda")

    def advance(oob):
        pos = dev(2, S - 1, 5)                       # row 1: three nodes behind the end of its cache; row 2: no cache row
        tree_advance([x[:, :, :1]], [x[:, :, 1:]], [kc], [vc], [ks], [vs], [False], par, tok, tok, pos, row_map=dev(0, 1, B), oob=oob)
        return pos

    def fork(oob):
        pos, starts = dev(4, 5, 6), dev(0, 0, 0)
        kv_fork([kc], [vc], [ks], [vs], [False], dev(0, 0, -1), dev(1, B, 2), pos, starts, oob=oob)
        return pos

    for call, skipped in ((advance, 2 * 3 + 2 * T), (fork, 2)):
        plain, watched = new(), new()
        want = call(plain)
        with Watch():
            got = call(watched)
            call(None)
        assert torch.equal(got, want) and int(plain) == int(watched) == skipped


def test_indexes_of_any_integer_type():
    from ultraviolet_b200.kernels import adjust_logits, tree_positions
    x = torch.randn((2, 100), generator=_gen(1), device="cuda")
    ids, bias = torch.tensor([3, 90, 3, 99], device="cuda"), torch.tensor([1.0, -2.0, 5.0, 0.5], device="cuda")
    want = adjust_logits(x, bias_ids=ids.int(), bias=bias)
    assert not torch.equal(want, adjust_logits(x))
    for dtype in (torch.int64, torch.int16, torch.int8, torch.uint8):
        assert torch.equal(adjust_logits(x, bias_ids=ids.to(dtype), bias=bias), want), dtype
    far = torch.tensor([3, 90, 3, 2 ** 40], device="cuda")
    assert torch.equal(adjust_logits(x, bias_ids=far, bias=bias)[:, :99], want[:, :99])
    par, pos = torch.tensor([-1, 0, 1, 0, -2], device="cuda"), torch.tensor([10, 20], device="cuda")
    for dtype in (torch.int64, torch.int32, torch.int16, torch.int8):
        assert tree_positions(par.to(dtype), pos.to(torch.int16)).tolist() == [[10, 11, 12, 11, 10], [20, 21, 22, 21, 20]], dtype
    # unsigned parents name no root: every node is absent
    assert tree_positions(torch.tensor([0, 0, 255], dtype=torch.uint8, device="cuda"), pos).tolist() == [[10] * 3, [20] * 3]


@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("B", [1, 2])
def test_rows_of_an_odd_pitch(B, T):
    """Slices of buffers whose rows are no multiple of 16 bytes: where one row or node is left of them, its dimension still has that stride."""
    from ultraviolet_b200.kernels import kv_fork, tree_advance, tree_attention
    S = 24
    x = torch.randn((B, T, 10, 64), generator=_gen(T), device="cuda").to(torch.bfloat16)
    kc, vc, ks, vs = _state(B, 1, S, 64, torch.bfloat16, 3)
    rows = torch.zeros((3, T * 640 + 3), dtype=torch.bfloat16, device="cuda")[:, :T * 640].unflatten(1, (T, 10, 64))[:B]
    nodes = torch.zeros((T + 1, 3, 645), dtype=torch.bfloat16, device="cuda")[..., :640].unflatten(2, (10, 64))[:T, :B].transpose(0, 1)
    assert rows.stride(0) % 8 and nodes.stride(1) % 8
    par, pos, zero = torch.arange(-1, T - 1, device="cuda"), torch.full((B,), 9, device="cuda"), torch.zeros(B, dtype=torch.long, device="cuda")
    tok = torch.zeros((B, T), dtype=torch.long, device="cuda")
    # and caches of which the same holds
    wide = [torch.zeros((3, S * 64 + e), dtype=torch.int8, device="cuda")[:, :S * 64].unflatten(1, (1, S, 64))[:B] for e in (5, 9)]
    wide[0].copy_(kc), wide[1].copy_(vc)
    caches = [(kc, vc)] + ([tuple(wide)] if B == 1 else [])       # (rows of a cache that follow each other have to be aligned)
    outs, ends = [], []
    for src in (x, rows.copy_(x), nodes.copy_(x)):
        for k, v in caches:
            outs.append(tree_attention(src[:, :, :8], src[:, :, 8:9], src[:, :, 9:], k, v, pos, zero, par, 0.2, k_scale=ks, v_scale=vs))
    for src in (x, rows, nodes):
        for k, v in caches:
            k[:, :, 9:9 + T], v[:, :, 9:9 + T] = 0, 0
            tree_advance([src[:, :, 8:9]], [src[:, :, 9:]], [k], [v], [ks], [vs], [False], par, tok, tok, pos.clone())
            ends.append((k.clone(), v.clone()))
            kv_fork([k], [v], [ks], [vs], [False], zero[:1], zero[:1], pos, zero)
    assert all(torch.equal(o, outs[0]) for o in outs)
    assert all(torch.equal(a, b) for e in ends for a, b in zip(e, ends[0])) and ends[0][0][:, :, 9:9 + T].abs().sum() > 0


def test_watched_logits_refuse_the_same_outputs():
    from torch.utils._python_dispatch import TorchDispatchMode
    from ultraviolet_b200.kernels import adjust_logits

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x = torch.randn((2, 40), generator=_gen(1), device="cuda")
    wrong = [torch.zeros(s, dtype=d, device="cuda") for s, d in (((3, 2, 40), torch.float32), ((1, 2, 40), torch.float32), ((2, 40), torch.int32),
                                                                ((2, 40), torch.float64), ((2, 41), torch.float32))]
    right = torch.zeros((2, 40), dtype=torch.float16, device="cuda")
    for out in wrong:
        with pytest.raises(ValueError):
            adjust_logits(x, out=out)
        with Watch(), pytest.raises(ValueError):
            adjust_logits(x, out=out)
        assert (out == 0).all()
    with Watch():
        assert adjust_logits(x, out=right) is right
    assert torch.equal(right, x.half())


def _exact(q, k, v, kc, vc, ks, vs, pos, parents, scale):
    """One row in 64 bits, starts 0: the mean of the values and of their magnitudes, (T, H, hd) each."""
    from oracle import kv as okv
    T, H, hd = q.shape
    keys, vals = [], []
    for x, c, s, to in ((k, kc, ks, keys), (v, vc, vs, vals)):
        codes, scales = (torch.from_numpy(a).to(q.device).double() for a in okv.quantize_kv(x.float().cpu().numpy()))     # (T, K, hd), (T, K)
        to += [torch.cat([c[:, :pos].double() * s[:, :pos, None].double(), (codes * scales[..., None]).transpose(0, 1)], 1)]
    keys, vals = keys[0], vals[0]                                                           # (K, pos + T, hd)
    G = H // keys.size(0)
    up = [ot.path_up(parents, t) for t in range(T)]
    s = torch.einsum("tkgd,knd->ktgn", q.double().view(T, -1, G, hd), keys) * scale
    for t in range(T):
        hidden = torch.ones(T, dtype=torch.bool, device=q.device)
        hidden[up[t]] = False
        s[:, t, :, pos:].masked_fill_(hidden, float("-inf"))
    w = torch.softmax(s, -1)
    there = torch.tensor([len(u) > 0 for u in up], device=q.device)[:, None, None]
    mean = lambda x: torch.einsum("ktgn,knd->tkgd", w, x).reshape(T, H, hd) * there
    return mean(vals), mean(vals.abs())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("route", sorted(ROUTES))
def test_attention_within_what_its_roundings_leave(route, dtype):
    """Half an ulp of the output; a weight times its value's scale is rounded to 11 bits, so that the mean moves by up to 2**-11 of
    A = sum w |V| / sum w, and scores of 32 .. 128 exact products summed in 32 bits move it by less than as much again; what is
    rounded below fp16's smallest normal is off by at most 2**-25 of the largest contribution a key, all of it below N 2**-25 max A."""
    B, T, H, K, hd, S, splits = ROUTES[route]
    run, x, ks, vs, pos, par = _call(route, dtype, "padded")
    got = run(x)
    kc, vc = _state(B, K, S, hd, dtype, T)[:2]
    for b in (0, B - 1):
        q, k, v = x[b].split([H, K, K], 1)
        ref, size = _exact(q, k, v, kc[b], vc[b], ks[b], vs[b], int(pos[b]), par[b].tolist(), 0.14)
        bound = 1.01 * UNIT[dtype] * 2 * ref.abs() + 2.0 ** -10 * size + S * 2.0 ** -25 * size.max() + 1e-7
        err = (got[b].double() - ref).abs()
        assert (err <= bound).all(), float((err / bound).max())
