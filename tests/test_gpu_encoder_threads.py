"""Embedding, gated feed-forward block and Newton-Schulz steps called from several threads at once, each on a stream of its own: the steps' launches, whose blocks wait for each other, stand in
each other's way on the SMs and still all finish; every call's result is looked at."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _together(jobs, rounds):
    """Every job's results of `rounds` calls, made by a thread of its own on its own stream."""
    results, errors, gate = [[] for _ in jobs], [], threading.Barrier(len(jobs))

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                gate.wait(30)
                for _ in range(rounds):
                    results[i].append(jobs[i]())
            stream.synchronize()
        except Exception as e:                                              # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors, errors
    torch.cuda.synchronize()
    return results


def _flat(x):
    return [x] if isinstance(x, torch.Tensor) else [t for y in x for t in _flat(y)]


def test_all_at_once():
    from haste_b200 import _lib
    from haste_b200.embedding import embedding_backward, embedding_forward
    from haste_b200.feedforward import gated_backward, gated_forward
    from haste_b200.optim import orthogonalize
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).cuda()
    ids, table, dy = torch.randint(0, 700, (5000,), generator=gen).cuda(), r(700, 96), r(5000, 96)
    x, wg, wu, wd, g = r(600, 256).to(BF), (0.06 * r(512, 256)).to(BF), (0.06 * r(512, 256)).to(BF), (0.04 * r(256, 512)).to(BF), r(600, 256).to(BF)
    one, many, large = [r(512, 768)], [r(40 + i, 300) for i in range(12)], [r(1024, 1024) for _ in range(8)]
    torch.cuda.synchronize()

    def block():
        y, gate, up = gated_forward(x, wg, wu, wd, keep=True)
        return (y, *gated_backward(g, x, wg, wu, wd, gate, up))

    jobs = [lambda: orthogonalize(one), lambda: orthogonalize(many), lambda: orthogonalize(large), block, lambda: (embedding_forward(ids, table), embedding_backward(dy, ids, 700))]
    want = [_flat(job()) for job in jobs]
    torch.cuda.synchronize()
    for got, expected in zip(_together(jobs, 12), want):
        assert len(got) == 12
        for result in got:
            assert all(torch.equal(a, b) for a, b in zip(_flat(result), expected))
    assert _lib.lib.haste_poll_status() == _lib.OK


def test_steps_at_once():
    from haste_b200 import _lib
    from haste_b200.optim import moment_offsets, muon_step
    shapes = [(300, 200), (128, 512), (700, 64)]

    def state(seed):
        gen = torch.Generator().manual_seed(seed)
        return [torch.randn(s, generator=gen).to(BF).cuda() for s in shapes], [torch.randn(s, generator=gen).cuda() for s in shapes], torch.zeros(moment_offsets([a * b for a, b in shapes])[-1], device="cuda")

    def steps(w, g, m):
        for t in range(1, 6):
            muon_step(w, g, m, step=t)
        return [*w, m]

    want = []
    for seed in range(3):
        want.append([t.clone() for t in steps(*state(seed))])
    states = [state(seed) for seed in range(3)]
    torch.cuda.synchronize()
    for got, expected in zip(_together([lambda s=s: steps(*s) for s in states], 1), want):
        assert all(torch.equal(a, b) for a, b in zip(got[0], expected))
    assert _lib.lib.haste_poll_status() == _lib.OK
