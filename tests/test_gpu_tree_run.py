"""GPU: the tree calls together, as a serving loop uses them: the example's model against the
same model token by token, a step in a graph, on other streams and devices."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

import axiom_amd
from axiom_amd.tree import latent_tree_decode_workspace_bytes
from test_gpu_tree_cache import case
from test_gpu_tree_verify import case as verify_case
from tree_testutil import step_inputs, trees

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "draft_tree.py"
    spec = importlib.util.spec_from_file_location("draft_tree", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_greedy_answer_is_the_one_token_by_token(cuda, example):
    steps, said, behind = example.run(device=cuda)
    assert steps >= 1 and all(len(s) >= 12 + steps for s in said)
    assert sum(map(len, said)) > 3 * (13 + steps)       # longer paths than place 0 were kept
    # fp32 throughout: two layers of 1e-5 each and products of 256 terms (1e-6), scores up to
    # about 10, and two of them are compared: 2 * 10 * 3e-5 where nothing amplifies an error
    assert max(behind) <= 6e-4


def test_sampled_answer_runs(cuda, example):
    steps, said, behind = example.run(n_new=30, sample=True, device=cuda)
    assert steps >= 1 and all(len(s) >= 12 + steps for s in said)
    assert all(0 <= t < example.VOCAB for s in said for t in s)


def start(example, device, B=3):
    """A prompt done, and a tree for the step after it."""
    torch.manual_seed(3)
    a = example.Answer(example.Model(device), B, 200)
    a.table = torch.arange(a.table.numel(), device=device).int().flip(0).view_as(a.table)
    prompt = torch.randint(example.VOCAB, (B, 40), device=device) % 9     # few tokens: every draft is there
    first = a.prompt(prompt).argmax(-1)
    drafted = [example.draft(p.tolist() + [int(t)]) for p, t in zip(prompt, first)]
    tokens = torch.tensor([t for t, _ in drafted], device=device)
    return a, tokens, torch.tensor([p for _, p in drafted], dtype=torch.int32, device=device)


def memory(a):
    return [a.state, a.conv, a.cache, a.lens]


@pytest.mark.parametrize("sample", [False, True])
def test_step_in_a_graph(cuda, example, sample):
    a, tokens, parents = start(example, cuda)
    N = tokens.shape[1]
    uniforms = torch.rand(3, N + 1, device=cuda) if sample else None
    before = [t.clone() for t in memory(a)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step(tokens, parents, uniforms)
    torch.cuda.current_stream().wait_stream(side)

    def reset():
        for t, x in zip(memory(a), before):
            t.copy_(x)

    def eager():
        reset()
        got = [t.clone() for t in a.step(tokens, parents, uniforms)]
        return got + [t.clone() for t in memory(a)]

    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a.step(tokens, parents, uniforms)
    for replay in range(4):
        if replay == 2:          # other drafts and numbers in the same buffers
            tokens.copy_(tokens.roll(1, 0))
            parents.copy_(trees(["random", "broken", "deep"], N, cuda, seed=5).where(torch.arange(N, device=cuda) > 0, -1))
            if sample:
                uniforms.copy_(torch.rand(3, N + 1, device=cuda))
        want = eager()
        reset()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip([*out, *memory(a)], want):
            assert torch.equal(x, y), replay


def calls(device, seed=0):
    """Every operator once on inputs of its own; returns a function that gives all outputs."""
    x = step_inputs(3, 20, 2, 128, "bf16", device, seed=seed)
    p = trees(["random", "chain", "broken"], 20, device, seed=seed)
    last = torch.tensor([13, 19, 4], dtype=torch.int32, device=device)
    q, cache, table, lens = case([700, 90, 20], 20, 4, 512, 64, 16, "bf16", device, seed=seed)
    sample = verify_case(["random", "chain", "star"], 9, 5003, "bf16", device, seed=seed)

    def run():
        out = []
        o, u = axiom_amd.kda_tree_step(*(x[n] for n in ("q", "k", "v", "g", "beta")), p, x["state"])
        out += [o, u, axiom_amd.kda_tree_commit(x["k"], x["g"], u, p, last, x["state"].clone())]
        out += axiom_amd.latent_tree_decode(q, cache, table, lens, p, 0.07)
        moved = cache.nan_to_num()
        out += [axiom_amd.latent_tree_commit(moved, table, lens, p, last), moved]
        return out + list(axiom_amd.tree_verify(*sample[:3])) + list(axiom_amd.tree_verify(*sample))

    return run


def test_another_stream_and_two_at_once(cuda):
    runs = [calls(cuda, seed) for seed in (1, 2)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for r, s in zip(runs, streams):      # nothing waits between them
            with torch.cuda.stream(s):
                got.append(r())
        torch.cuda.synchronize()
        for w, x in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(w, x))


def test_inputs_of_the_same_stream_are_waited_for(cuda):
    """Inputs written by work that is still queued on the call's stream."""
    a = torch.randn(4096, 4096, device=cuda)
    x = step_inputs(2, 9, 2, 128, "fp32", cuda, seed=3)
    p = trees(["random", "chain"], 9, cuda)
    o, _ = axiom_amd.kda_tree_step(*(x[n] for n in ("q", "k", "v", "g", "beta")), p, x["state"])
    s = torch.cuda.Stream()
    late = {n: torch.zeros_like(t) for n, t in x.items()}
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(4):
            a = a @ a * 1e-3
        for n, t in x.items():
            late[n].copy_(t)
        got, _ = axiom_amd.kda_tree_step(*(late[n] for n in ("q", "k", "v", "g", "beta")), p, late["state"])
    torch.cuda.synchronize()
    assert torch.equal(o, got)


def test_one_workspace_for_successive_calls(cuda):
    """A workspace of the largest call serves smaller ones after it, whatever they left in it."""
    cases = [([900, 33, 64], 20, 4), ([5000, 17, 12], 5, 16), ([40, 300, 9], 9, 1)]
    need = max(latent_tree_decode_workspace_bytes(3, N, H, 512, 64, 16, -(-max(lens) // 16)) for lens, N, H in cases)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=cuda)
    for i, (lens, N, H) in enumerate(cases * 2):
        q, cache, table, n = case(lens, N, H, 512, 64, 16, "bf16", cuda, seed=i)
        p = trees(["random", "broken", "chain"], N, cuda, seed=i)
        want = axiom_amd.latent_tree_decode(q, cache, table, n, p, 0.07)
        got = axiom_amd.latent_tree_decode(q, cache, table, n, p, 0.07, workspace=ws)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_another_device(cuda):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    other = torch.device("cuda:1")
    got = calls(other, 4)()              # the current device stays 0
    torch.cuda.synchronize(other)
    with torch.cuda.device(other):
        want = calls(other, 4)()
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
