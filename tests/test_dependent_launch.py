"""Kernels that may be launched while their predecessor on the stream still runs: each has to wait for it before it reads anything."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ultraviolet_b200", "csrc")


def _sources():
    for n in sorted(os.listdir(CSRC)):
        if n.endswith((".cu", ".cuh")) and n != "common.cuh":
            with open(os.path.join(CSRC, n)) as f:
                yield n, re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def _block(text, at):
    """The block that opens at or behind position at."""
    at = text.index("{", at)
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError("a block without an end")


def _kernels():
    """name -> body of every kernel."""
    out = {}
    for _, text in _sources():
        for m in re.finditer(r"__global__", text):
            end = text.index("{", m.end())
            head = re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", text[m.end():end])
            out[re.search(r"(\w+)\s*\(", head).group(1)] = _block(text, end)
    return out


def _launched_early(kernels):
    """Kernels that are handed to a launch with the programmatic attribute, by name or as the variable `kern` set before it."""
    names = set()
    for _, text in _sources():
        for m in re.finditer(r"\blaunch_(?:pdl|cluster|cluster_pdl)\s*\(", text):
            words = re.findall(r"\w+", text[m.end():m.end() + 200])
            name = next(w for w in words if w == "kern" or w in kernels)
            names.add(re.findall(r"\bkern = (\w+)", text[:m.start()])[-1] if name == "kern" else name)
    return names


def test_every_kernel_that_may_start_early_waits():
    kernels = _kernels()
    early = _launched_early(kernels)
    assert {"tree_rows_kernel", "tree_tc_merge_kernel", "sample_kernel", "attn_split_kernel", "prefill_attn_kernel"} <= early, early
    assert not sorted(k for k in early if "pdl_wait()" not in kernels[k])


STEP = """
import sys, hashlib, numpy as np, torch
from tests.test_drafted_gpu import SPECS, _model, _prefilled
m = _model("uv50m")
V = m.cfg.vocab_size
st = _prefilled(m, np.random.default_rng(0).integers(1, V, (3, 20)), np.zeros(3, np.int64), 200)
parents = torch.tensor([-1, 0, 1, 0, 3], device="cuda", dtype=torch.int32)
g, h = torch.Generator(device="cuda").manual_seed(1), hashlib.sha256()
for _ in range(12):
    tok = torch.randint(0, V, (3, 5), generator=g, device="cuda")
    h.update(m.tree_step(tok, parents, st).cpu().numpy().tobytes())
    target = tok[:, [1, 2, 0, 4, 0]].clone()
    m.tree_accept(tok, target, parents, st)
    h.update(st.pos.cpu().numpy().tobytes())
for y in (st.k, st.v):
    for t in y:
        h.update(t.contiguous().cpu().numpy().tobytes())
m.engine.check_status()
print(h.hexdigest())
"""


@pytest.mark.gpu
def test_tree_steps_are_the_same_with_dependent_launches():
    out = []
    for pdl in ("0", "1"):
        env = {**os.environ, "UVDECODE_PDL": pdl, "PYTHONPATH": ROOT}
        got = subprocess.run([sys.executable, "-c", STEP], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
        assert got.returncode == 0, got.stderr[-2000:]
        out.append(got.stdout.split()[-1])
    assert out[0] == out[1]


def test_tree_kernels_that_give_up_wait_for_what_is_under_way():
    """A kernel whose wait has run out ends behind its own copies and products, by another bounded wait: what arrives later would land in
    the shared memory, or the tensor memory, of whoever has it then."""
    kernels = _kernels()
    rows, tc = kernels["tree_rows_kernel"], kernels["tree_tc_kernel"]
    assert re.search(r"if \(lost && producer && lane == 0\) drain_copies\(full, issued\)", rows[rows.index("lost = s_dead"):])
    end = tc[tc.rindex("__syncthreads()"):]
    commit, wait, free = (end.index(x) for x in ("tc_commit(tc_smem_u32(&sh.drained))", "tc_mbar_wait(tc_smem_u32(&sh.drained)", "tcgen05.dealloc"))
    assert commit < wait < free
    with open(os.path.join(CSRC, "tree_attn_tc.cu")) as f:      # the codes come by cp.async, which each thread waits for
        body = f.read()
    convert = body[body.index("void convert_tiles"):body.index("void mask_scores")]
    assert convert.rstrip().rindex("cp.async.wait_all") > convert.rindex("mbar_arrive_one")
