"""Embedding, layer norm, gated feed-forward block and the fused step of projection, norm and sparse layer, trained by Muon and AdamW: one run of them together, as an encoder in front of the
sparse layer uses them, against the same composition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import encoder_oracle as eo

BF = torch.bfloat16


class _Encoder(torch.nn.Module):
    def __init__(self, vocab, width, hidden):
        super().__init__()
        from haste_b200.embedding import Embedding
        from haste_b200.feedforward import GatedFeedForward
        from haste_b200.norm import LayerNorm
        self.tokens = Embedding(vocab, width, padding_idx=0, device="cuda", dtype=BF)
        self.norm = LayerNorm(width, device="cuda")
        self.block = GatedFeedForward(width, hidden, device="cuda")

    def forward(self, ids):
        e = self.tokens(ids)
        e = e + self.block(self.norm(e))
        keep = (ids != 0).to(BF)[..., None]
        return (e * keep).sum(1) / keep.sum(1).clamp(min=1)


def _setup(seed=0):
    from haste_b200.norm import LayerNorm
    torch.manual_seed(seed)
    enc = _Encoder(500, 128, 256)
    lin, norm = torch.nn.Linear(128, 64, device="cuda", dtype=BF), LayerNorm(64, device="cuda")
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(1, 500, (24, 30), generator=gen)
    for i in range(24):
        ids[i, 30 - i:] = 0                                                 # a padded batch; the last texts are nearly empty
    ids[5] = 0                                                              # and one is empty
    return enc, lin, norm, ids.cuda()


def _exact_features(enc, ids, table, wg, wu, wd, g, b):
    e = table[ids]
    mean, var = e.mean(-1, keepdim=True), e.var(-1, keepdim=True, unbiased=False)
    n = (e - mean) / (var + enc.norm.eps).sqrt() * g + b
    gate = n @ wg.t()
    e = e + (gate * torch.sigmoid(gate) * (n @ wu.t())) @ wd.t()
    keep = (ids != 0).double()[..., None]
    return (e * keep).sum(1) / keep.sum(1).clamp(min=1)


def test_gradients_of_the_run():
    enc, _, _, ids = _setup()
    w = torch.randn(24, 128, device="cuda")
    (enc(ids).float() * w).sum().backward()
    leaves = [enc.tokens.weight, enc.block.w_gate, enc.block.w_up, enc.block.w_down, enc.norm.weight, enc.norm.bias]
    exact = [p.detach().double().requires_grad_() for p in leaves]
    (_exact_features(enc, ids, *exact) * w.double()).sum().backward()
    for name, p, q in zip(("table", "w_gate", "w_up", "w_down", "norm.weight", "norm.bias"), leaves, exact):
        got, want = p.grad.double(), q.grad.clone()
        if name == "table":
            want[0] = 0
            assert not got[0].any()
        # about ten roundings to bf16 lie on the way, each 2^-8 at most of what it rounds, and none is amplified by more than the norm's and the block's slopes (two or so)
        assert float((got - want).norm()) <= 20 * 2 ** -8 * float(want.norm()), name


def test_training_steps():
    """Encoder, projection, norm and sparse layer with Muon over the matrices and AdamW over the rest: every parameter moves as its optimizer says."""
    from haste_b200.fused import FusedFFIShard
    from haste_b200.optim import AdamW, Muon
    from haste_b200.projected import ProjectedFusedStep
    from oracle import ffi_oracle as fo
    enc, lin, norm, ids = _setup(1)
    inp = fo.make_inputs(24, 64, 500, 32, 32, 5, 1.1, seed=3, x_kind="normal")
    shard = FusedFFIShard(inp["loc"].cuda(), inp["W"].clone().cuda(), inp["bias"].clone().cuda(), 32, 64, loss="bce", lr=0.05, weight_decay=0.0, seed=42)
    matrices = [enc.block.w_gate, enc.block.w_up, enc.block.w_down, lin.weight]
    rest = [enc.tokens.weight, enc.norm.weight, enc.norm.bias, lin.bias, norm.weight, norm.bias]
    muon, adam = Muon(matrices, lr=1e-2, adjust="match_rms_adamw"), AdamW(rest, lr=1e-3, weight_decay=0.0)
    step = ProjectedFusedStep(lin, norm, shard, [muon, adam])
    for t in range(3):
        muon.zero_grad()
        adam.zero_grad()
        before = [p.detach().clone() for p in matrices + rest]
        h = enc(ids)
        dh, loss = step.backward(h.detach(), inp["targets"].cuda())
        h.backward(dh)
        momentum = [muon.state[p]["momentum_buffer"].clone() if p in muon.state else torch.zeros(p.shape, device="cuda") for p in matrices]
        step.update()
        assert torch.isfinite(loss).all()
        for p, old, m in zip(matrices, before, momentum):
            new = 0.95 * m.double() + 0.05 * p.grad.double()
            u = 0.95 * new + 0.05 * p.grad.double()
            x, tol = eo.orthogonalize_bound(u)
            rate = eo.muon_rate(p.shape, 1e-2, "match_rms_adamw")
            want = old.double() * (1 - 1e-2 * 0.1) - rate * x
            # weights are rounded stochastically: a whole step of bf16, 2^-7, at most
            assert float((p.double() - want).norm()) <= rate * tol + 2 ** -7 * float(want.norm())
        assert all(not torch.equal(p, old) for p, old in zip(rest, before[len(matrices):]))
        assert torch.equal(enc.tokens.weight[0], before[len(matrices)][0])      # the padding row has no gradient


def test_step_in_a_graph():
    """Forward and backward of the run captured and replayed beside the eager ones (backward passes by the kernels' functions, without an eager graph of the same leaves)."""
    from haste_b200 import embedding, feedforward, norm as ln
    enc, _, _, ids = _setup(2)
    table, wg, wu, wd = (p.detach() for p in (enc.tokens.weight, enc.block.w_gate, enc.block.w_up, enc.block.w_down))
    g, b = enc.norm.weight.detach(), enc.norm.bias.detach()
    dy = torch.randn(24, 30, 128, device="cuda").to(BF)

    def run():
        e = embedding.embedding_forward(ids, table)
        n, mean, rstd = ln.layer_norm_forward(e, g, b)
        y, gate, up = feedforward.gated_forward(n, wg, wu, wd, keep=True)
        dn, dwg, dwu, dwd = feedforward.gated_backward(dy, n, wg, wu, wd, gate, up)
        de, dg, db = ln.layer_norm_backward(dn, e, g, mean, rstd)
        return y, dwg, dwu, dwd, dg, db, embedding.embedding_backward(de, ids, 500, 1.0, 0)

    want = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for t in out:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(out, want))
