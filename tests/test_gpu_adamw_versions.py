"""AdamW writes parameters by address; autograd has to learn of it as of any other change in place."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_step_between_forward_and_backward_is_an_error(dtype, bits):
    from haste_b200.optim import AdamW
    layer = torch.nn.Linear(64, 32, device="cuda", dtype=dtype)
    opt = AdamW(layer.parameters(), state_bits=bits)
    x = torch.randn(4, 64, device="cuda", dtype=dtype, requires_grad=True)
    layer(x).sum().backward()
    y = layer(x)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    layer(x).sum().backward()                                               # a new graph is fine


def test_what_counts_as_written():
    from haste_b200.optim import Quantized, adamw_step, moment_offsets
    sizes = [300, 20, 7]
    n = moment_offsets(sizes)[-1]
    p, g = [torch.zeros(s, device="cuda") for s in sizes], [torch.ones(300, device="cuda"), None, torch.ones(7, device="cuda")]
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    before = [t._version for t in p + [m, v]]
    adamw_step(p, g, m, v, step=1)
    assert [t._version - b for t, b in zip(p + [m, v], before)] == [1, 0, 1, 1, 1]
    m, v = (Quantized(torch.zeros(n, device="cuda", dtype=torch.uint8), torch.zeros(n // 256, device="cuda"), s) for s in (True, False))
    parts = (m.codes, m.scales, v.codes, v.scales)
    was = [t._version for t in parts]
    adamw_step(p, g, m, v, step=1)
    assert [t._version - b for t, b in zip(parts, was)] == [1] * 4
    with pytest.raises(RuntimeError):
        adamw_step(p, g, m, v, step=0)
    assert p[0]._version == before[0] + 2                                   # a refused call has written nothing
    with torch.inference_mode():                                            # tensors without a counter
        q, h = [torch.zeros(8, device="cuda")], [torch.ones(8, device="cuda")]
        adamw_step(q, h, torch.zeros(256, device="cuda"), torch.zeros(256, device="cuda"), step=1)
        assert bool((q[0] < 0).all())
