"""A small hybrid model (a KDA layer, a latent layer) that answers with drafted trees.

    python examples/draft_tree.py

Every step drafts a tree of N places a sequence, runs the model over all of them
at once, keeps the path that the model itself would have said, and moves states and
caches there.  Place 0 is the token that the step before drew: its row of the target
is that token alone, so it is always kept.  The other places hold what followed the
same token earlier in the sequence, the newest and the one before it; a token without
a successor leaves its places without a draft.  The draft is sure of its tokens, so
``tree_verify`` needs no draft distributions, and the answer is one of the model's own:
greedily the one that :func:`one_by_one` gives, token by token.
"""

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from axiom_amd import (kda_epilogue, kda_prologue, kda_recurrent_step, kda_tree_commit, kda_tree_step,  # noqa: E402
                       latent_append, latent_decode, latent_tree_commit, latent_tree_decode, tree_verify)

VOCAB, DM, H, D, K, DN, DR, R, PAGE = 96, 256, 4, 128, 4, 64, 32, 256, 16
SCALE = (DN + DR) ** -0.5
PARENTS = [-1, 0, 0, 1, 1, 2, 3, 6]      # place 0, two successors of it, two of the first's, ...
RANK = [-1, 0, 1, 0, 1, 0, 0, 0]         # which of its parent's successors a place holds


class Model:
    def __init__(self, device="cuda", positions=512, seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape):
            return torch.randn(*shape, device=device, generator=gen) * shape[0] ** -0.5

        self.embed = torch.randn(VOCAB, DM, device=device, generator=gen)
        self.wqkv = weight(3, DM, H * D) * (3 / DM) ** 0.5
        self.taps = weight(3, K, H * D)
        self.wg, self.wb, self.wz, self.wo = weight(DM, H * D), weight(DM, H), weight(DM, H * D), weight(H * D, DM)
        self.lq, self.ld = weight(DM, H * (DN + DR)), weight(DM, R + DR)
        self.norm = torch.ones(R, device=device)
        self.lk, self.lv = weight(H, DN, R) * (H / DN) ** 0.5, weight(H, R, DN) * (H / R) ** 0.5
        self.lo, self.unembed = weight(H * DN, DM), weight(DM, VOCAB)
        inv = 10000.0 ** (-torch.arange(0, DR, 2, device=device) / DR)
        a = torch.arange(positions, device=device)[:, None] * inv
        self.cos_sin = torch.cat([a.cos(), a.sin()], -1)

    def kda_inputs(self, x, windows):
        """windows [3, M, K, H*D]: the conv's inputs up to each of x's M tokens, the newest last."""
        M = x.shape[0]
        q, k, v, _ = kda_prologue(*windows, *self.taps, H, return_state=False, out_dtype=torch.float32)
        q, k, v = (t[:, -1].contiguous() for t in (q, k, v))
        g = -torch.nn.functional.softplus(x @ self.wg).view(M, H, D)
        return q, k, v, g, torch.sigmoid(x @ self.wb)

    def kda_output(self, x, o):
        M = x.shape[0]
        y = kda_epilogue(o.reshape(M, 1, H, D), (x @ self.wz).view(M, 1, H * D), out_dtype=torch.float32)
        return x + y.view(M, H * D) @ self.wo

    def latent_query(self, x, positions, slots, cache):
        """The tokens' rows into the cache; their queries in the absorbed form [M, H, R + DR]."""
        M = x.shape[0]
        q = (x @ self.lq).view(M, H, DN + DR)
        qa = torch.empty(M, H, R + DR, device=x.device)
        latent_append(x @ self.ld, positions, slots, self.cos_sin, cache, self.norm, 1e-6, q[..., DN:], qa[..., R:])
        qa[..., :R] = torch.bmm(q[..., :DN].transpose(0, 1).contiguous(), self.lk).transpose(0, 1)
        return qa

    def scores(self, x, o):
        M = x.shape[0]
        o = torch.bmm(o.reshape(M, H, R).transpose(0, 1).contiguous(), self.lv)
        return (x + o.transpose(0, 1).reshape(M, H * DN) @ self.lo) @ self.unembed


class Answer:
    """B sequences in progress: KDA states, conv inputs, the latent cache, lengths."""

    def __init__(self, model, B, max_len):
        dev = model.embed.device
        self.m, self.B, self.dev = model, B, dev
        self.state = torch.zeros(B, H, D, D, device=dev)
        self.conv = torch.zeros(3, B, K - 1, H * D, device=dev)
        pages = -(-max_len // PAGE)
        self.cache = torch.zeros(B * pages, PAGE, R + DR, device=dev)
        self.table = torch.randperm(B * pages, device=dev).int().view(B, pages)     # pages in any order
        self.lens = torch.zeros(B, dtype=torch.int32, device=dev)
        self.rows = torch.arange(B, device=dev)

    def slots(self, rows):
        return self.table.long().gather(1, rows // PAGE) * PAGE + rows % PAGE

    def forward(self, tokens, parents):
        """The model over the places: scores [B, N, VOCAB]; keeps what :meth:`keep` needs."""
        m, (B, N) = self.m, tokens.shape
        x = m.embed[tokens.clamp_min(0).reshape(-1)]
        # what precedes a place among the sequence's last K - 1 conv inputs and the places' own
        inputs = torch.cat([self.conv, torch.matmul(x, m.wqkv).view(3, B, N, H * D)], 2)
        up = torch.where(parents < 0, K - 2, parents + K - 1).long()
        at = [torch.arange(K - 1, K - 1 + N, device=self.dev).expand(B, N)]
        for _ in range(K - 1):
            above = up.gather(1, (at[0] - (K - 1)).clamp_min(0))
            at.insert(0, torch.where(at[0] < K - 1, at[0] - 1, above).clamp_min(0))
        windows = inputs[:, self.rows[:, None, None], torch.stack(at, -1)].contiguous()
        q, k, v, g, beta = (t.view(B, N, *t.shape[1:]) for t in m.kda_inputs(x, windows.view(3, B * N, K, H * D)))
        o, u = kda_tree_step(q, k, v, g, beta, parents, self.state)
        self.new = k, g, u, windows
        x = m.kda_output(x, o)

        depth = torch.zeros(B, N, dtype=torch.int64, device=self.dev)
        for i in range(1, N):                                # a place comes after its parent
            p = parents[:, i].long()
            depth[:, i] = torch.where(p < 0, 0, depth[self.rows, p.clamp_min(0)] + 1)
        start = self.lens.long()[:, None]
        rows = self.slots(start + torch.arange(N, device=self.dev))
        qa = m.latent_query(x, (start + depth).reshape(-1), rows.reshape(-1), self.cache)
        o, _ = latent_tree_decode(qa.view(B, N, H, R + DR), self.cache, self.table, self.lens + N, parents, SCALE)
        return m.scores(x, o).view(B, N, VOCAB)

    def keep(self, parents, last):
        """The model's memory after the path of place last[b]."""
        k, g, u, windows = self.new
        kda_tree_commit(k, g, u, parents, last, self.state)
        kept = windows[:, self.rows, last.clamp_min(0).long(), 1:]
        self.conv.copy_(torch.where((last >= 0)[:, None, None], kept, self.conv))
        self.lens.copy_(latent_tree_commit(self.cache, self.table, self.lens + parents.shape[1], parents, last))

    def prompt(self, tokens):
        """A prompt [B, 1 .. 64] as a chain of places, all kept (the layers' chunked forms take long ones);
        the scores of its last token."""
        B, N = tokens.shape
        chain = torch.arange(-1, N - 1, dtype=torch.int32, device=self.dev).expand(B, N).contiguous()
        scores = self.forward(tokens, chain)
        self.keep(chain, torch.full((B,), N - 1, dtype=torch.int32, device=self.dev))
        return scores[:, -1]

    def step(self, tokens, parents, uniforms=None):
        """One tree; ``uniforms`` None: greedy.  Returns tree_verify's ``(last, next_token, accepted)``.

        Nothing is read back on the host: a fixed list of launches, fit for a graph.
        """
        scores = self.forward(tokens, parents)
        sure = torch.zeros(self.B, 1, VOCAB, device=self.dev).scatter_(2, tokens[:, :1, None], 1.0)
        target = torch.cat([sure, scores if uniforms is None else torch.softmax(scores, -1)], 1)
        verdict = tree_verify(target, tokens, parents, uniforms)
        self.keep(parents, verdict[0])
        return verdict


def draft(said):
    """Tokens and parents of a tree that begins with the last token said (host lists)."""
    seen = {}
    for a, b in zip(said, said[1:]):
        seen[a] = [b] + [c for c in seen.get(a, []) if c != b]
    tokens, parents = [said[-1]], list(PARENTS)
    for i in range(1, len(PARENTS)):
        after = seen.get(tokens[PARENTS[i]], [])
        tokens.append(after[RANK[i]] if len(after) > RANK[i] else -1)
        if tokens[i] < 0:
            parents[i] = -2
    return tokens, parents


def one_by_one(model, said, max_len):
    """Scores [len(said), VOCAB] of one sequence, a token at a time by the single-token operators."""
    a = Answer(model, 1, max_len)
    out = []
    for t, token in enumerate(said):
        x = model.embed[torch.tensor([token], device=a.dev)]
        window = torch.cat([a.conv, torch.matmul(x, model.wqkv).view(3, 1, 1, H * D)], 2)
        a.conv = window[:, :, 1:]
        x = model.kda_output(x, kda_recurrent_step(*model.kda_inputs(x, window), a.state))
        at = torch.tensor([t], device=a.dev)
        qa = model.latent_query(x, at, a.slots(at[:, None])[0], a.cache)
        o, _ = latent_decode(qa.view(1, 1, H, R + DR), a.cache, a.table, (at + 1).int(), SCALE)
        out.append(model.scores(x, o))
    return torch.cat(out)


def run(B=3, n_prompt=12, n_new=100, sample=False, device="cuda"):
    """Prompts, then trees until every sequence has n_new more tokens.

    Returns the steps taken, the tokens said and, per sequence, how far a said token's
    score lies below the best of its row when the sequence is run token by token.
    """
    torch.manual_seed(0)
    max_len = n_prompt + n_new + 2 * len(PARENTS)
    model = Model(device, max_len)
    said = torch.randint(VOCAB, (B, n_prompt)).tolist()
    a = Answer(model, B, max_len)
    scores = a.prompt(torch.tensor(said, device=device))
    first = torch.multinomial(torch.softmax(scores, -1), 1)[:, 0] if sample else scores.argmax(-1)
    for s, token in zip(said, first.tolist()):
        s.append(token)
    steps = 0
    while min(map(len, said)) < n_prompt + n_new and max(map(len, said)) + len(PARENTS) < max_len:
        trees = [draft(s) for s in said]
        tokens = torch.tensor([t for t, _ in trees], device=device)
        parents = torch.tensor([p for _, p in trees], dtype=torch.int32, device=device)
        uniforms = torch.rand(B, len(PARENTS) + 1, device=device) if sample else None
        last, after, _ = a.step(tokens, parents, uniforms)
        for s, (t, p), i, token in zip(said, trees, last.tolist(), after.tolist()):
            path = []
            while i > 0:                                     # place 0 has been said already
                path.append(t[i])
                i = p[i]
            s += path[::-1] + [token]
        steps += 1
    behind = []
    for s in said:
        scores = one_by_one(model, s, max_len)[n_prompt - 1:-1]
        token = torch.tensor(s[n_prompt:], device=device)
        behind.append(float((scores.max(-1).values - scores.gather(1, token[:, None])[:, 0]).max()))
    return steps, said, behind


if __name__ == "__main__":
    steps, said, behind = run()
    print(f"{steps} steps of {len(PARENTS)} places: {[len(s) - 13 for s in said]} tokens")
    print(f"greedy token's score below the best of the same sequence token by token: {max(behind):.1e}")
    steps, said, _ = run(sample=True)
    print(f"{steps} steps with samples: {[len(s) - 13 for s in said]} tokens")
