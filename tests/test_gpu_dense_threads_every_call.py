"""Dense operators from several host threads, each on its own stream: every single call gives what it gives alone."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def test_every_call_from_threads():
    from haste_b200 import optim
    from haste_b200.norm import layer_norm_backward, layer_norm_forward
    gen = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    calls = []
    for rows, D, dtype in ((300, 768, BF), (1700, 1000, F32), (4099, 1021, BF), (12, 9000, F32)):
        x, w, dy = rnd(rows, D).to(dtype), rnd(D), rnd(rows, D).to(dtype)

        def norm(x=x, w=w, dy=dy):
            y, mean, rstd = layer_norm_forward(x, w, w)
            return (y, *layer_norm_backward(dy, x, w, mean, rstd))
        calls.append(norm)
    for bits, sizes in ((32, [5000, 3, 700]), (8, [300] * 40), (8, [2000000])):
        n = optim.moment_offsets(sizes)[-1]
        p, g = [rnd(s) for s in sizes], [rnd(s) for s in sizes]

        def step(bits=bits, p=p, g=g, n=n):
            q = [t.clone() for t in p]
            m = [torch.zeros(n, device="cuda") for _ in range(2)]
            if bits == 8:
                m = [optim.quantize(t, s) for t, s in zip(m, (True, False))]
            norm = optim.adamw_step(q, g, *m, step=3, max_norm=1.0)
            return (*q, norm, *(m if bits == 32 else (m[0].codes, m[0].scales, m[1].codes, m[1].scales)))
        calls.append(step)
    want = [c() for c in calls]
    torch.cuda.synchronize()
    errors = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                wrong = torch.zeros((), device="cuda", dtype=torch.int64)
                for _ in range(60):
                    for a, b in zip(calls[k](), want[k]):
                        wrong += (a != b).sum()
                torch.cuda.current_stream().synchronize()
                assert int(wrong) == 0
        except BaseException as e:
            errors.append((k, e))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
