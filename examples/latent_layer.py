"""A latent-attention layer out of the package's operators: one training step,
a prompt into the paged cache, tokens decoded from it.

    python examples/latent_layer.py

The layer's parameters are the query projection, the down-projection to a latent
of R elements and a rotated key part of dr, the latent's norm, its up-projection
to keys and values, and the output projection; the projections are torch's
matrix products, the rest is ``latent_attn`` (expanded: training and the
prompt), ``latent_append`` and ``latent_decode`` (absorbed: single tokens).  The
decoded tokens are compared with the expanded form over the whole sequence.
"""

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from axiom_amd import latent_append, latent_attn, latent_attn_fwd, latent_decode  # noqa: E402

DM, H, DN, DR, R, PAGE, EPS = 512, 16, 128, 64, 512, 64, 1e-6
SCALE = (DN + DR) ** -0.5


def angles(n, device):
    """[n, DR] fp32: cosines of the DR/2 angles of positions 0 .. n - 1, then sines."""
    inv = 10000.0 ** (-torch.arange(0, DR, 2, device=device, dtype=torch.float32) / DR)
    a = torch.arange(n, device=device, dtype=torch.float32)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], -1)


def rotate(x, cs):
    """Rotation of x's last axis (pairs i, i + DR/2); cs broadcasts against it."""
    a, b = x.float().chunk(2, -1)
    c, s = cs.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


class LatentLayer(torch.nn.Module):
    def __init__(self, device="cuda", dtype=torch.bfloat16):
        super().__init__()

        def weight(n_in, n_out):
            return torch.nn.Parameter(torch.randn(n_in, n_out, device=device, dtype=dtype) * n_in ** -0.5)

        self.wq = weight(DM, H * (DN + DR))
        self.wd = weight(DM, R + DR)
        self.norm = torch.nn.Parameter(torch.ones(R, device=device))
        self.wu = weight(R, H * 2 * DN)          # a head's key, then its value
        self.wo = weight(H * DN, DM)

    def forward(self, x, cs):
        """Training form; x [B, T, DM], cs the angles of positions 0 .. T - 1."""
        B, T, _ = x.shape
        qn, qr = (x @ self.wq).view(B, T, H, DN + DR).split([DN, DR], -1)
        c, kr = (x @ self.wd).split([R, DR], -1)
        c = torch.nn.functional.rms_norm(c.float(), (R,), self.norm, EPS).to(x.dtype)
        q = torch.cat([qn, rotate(qr, cs[:, None])], -1)
        o = latent_attn(q, (c @ self.wu).view(B, T, H, 2 * DN), rotate(kr, cs))
        return o.reshape(B, T, H * DN) @ self.wo

    @torch.no_grad()
    def prompt(self, x, cs, cache, slots):
        """The prompt x [B, T, DM] into the cache at slots [B, T]; its outputs."""
        B, T, _ = x.shape
        q = (x @ self.wq).view(B * T, H, DN + DR)
        pos = torch.arange(T, device=x.device).repeat(B)
        qr = q[..., DN:]
        latent_append((x @ self.wd).view(B * T, R + DR), pos, slots.reshape(-1), cs, cache, self.norm, EPS, qr, qr)
        rows = cache.view(-1, R + DR)[slots]     # normed and rotated, as decoding will read them
        kv = (rows[..., :R] @ self.wu).view(B, T, H, 2 * DN)
        o, _ = latent_attn_fwd(q.view(B, T, H, DN + DR), kv, rows[..., R:])
        return o.reshape(B, T, H * DN) @ self.wo

    @torch.no_grad()
    def absorb(self):
        """The up-projection's halves as decoding uses them: [H, DN, R] and [H, R, DN]."""
        w = self.wu.view(R, H, 2, DN)
        return w[:, :, 0].permute(1, 2, 0).contiguous(), w[:, :, 1].permute(1, 0, 2).contiguous()

    @torch.no_grad()
    def decode(self, x, positions, slots, table, lens, cs, cache, absorbed):
        """One token a sequence; x [B, DM], lens counts it."""
        B = x.shape[0]
        wk, wv = absorbed
        q = (x @ self.wq).view(B, H, DN + DR)
        qa = torch.empty(B, 1, H, R + DR, device=x.device, dtype=x.dtype)
        latent_append(x @ self.wd, positions, slots, cs, cache, self.norm, EPS, q[..., DN:], qa[:, 0, :, R:])
        qa[:, 0, :, :R] = torch.bmm(q[..., :DN].transpose(0, 1).contiguous(), wk).transpose(0, 1)
        o, _ = latent_decode(qa, cache, table, lens, SCALE)
        o = torch.bmm(o[:, 0].transpose(0, 1).contiguous(), wv)          # [H, B, DN]
        return o.transpose(0, 1).reshape(B, H * DN) @ self.wo


def run(B=3, T_prompt=130, T_new=8, device="cuda"):
    """A training step, then prompt and decoding.  Returns the losses before and
    after the step, and the relative deviation of the prompt's and the decoded
    outputs from the expanded form's over the whole sequence."""
    torch.manual_seed(0)
    T = T_prompt + T_new
    layer, cs = LatentLayer(device), angles(T, device)
    x = torch.randn(B, T, DM, device=device, dtype=torch.bfloat16)
    target = torch.randn(B, T, DM, device=device)

    opt = torch.optim.SGD(layer.parameters(), lr=1.0)
    losses = []
    for _ in range(2):
        loss = (layer(x, cs).float() - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())

    with torch.no_grad():
        want = layer(x, cs).float()
    pages = (T + PAGE - 1) // PAGE
    cache = torch.zeros(B * pages, PAGE, R + DR, device=device, dtype=torch.bfloat16)
    table = torch.randperm(B * pages, device=device).to(torch.int32).view(B, pages)   # pages in any order
    tok = torch.arange(T, device=device)
    slots = table.long()[:, tok // PAGE] * PAGE + tok % PAGE
    got = torch.empty_like(want)
    got[:, :T_prompt] = layer.prompt(x[:, :T_prompt], cs, cache, slots[:, :T_prompt]).float()
    absorbed = layer.absorb()
    for t in range(T_prompt, T):
        now = torch.full((B,), t, device=device)
        lens = (now + 1).to(torch.int32)
        got[:, t] = layer.decode(x[:, t], now, slots[:, t].contiguous(), table, lens, cs, cache, absorbed).float()

    def deviation(a, b):
        return float((a - b).norm() / b.norm())

    return (losses, deviation(got[:, :T_prompt], want[:, :T_prompt]), deviation(got[:, T_prompt:], want[:, T_prompt:]))


if __name__ == "__main__":
    (before, after), prompt, decoded = run()
    print(f"loss {before:.4f} -> {after:.4f} after a step")
    print(f"deviation from the expanded form: prompt {prompt:.2e}, decoded {decoded:.2e}")
