"""The decoder operators inside sessions: what stands next to them, what order their runs keep, what is left when one fails, and
which graphs are refused."""
import math

import pytest

import decoder_oracle as D
import test_gpu_decoder as G

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ---- beside kernels that hold tensor memory ------------------------------------------------------
@pytest.mark.parametrize("sequences", [8, 900])
def test_prompts_in_front_of_a_small_product(sequences):
    """A prompt kernel of 64-lane heads leaves room on its SM for a block of the small product kernel behind it, which takes its
    tensor memory before it waits: the prompt's own must have been taken by then.  With hundreds of sequences the prompt kernel
    is still counting them when the other starts.  Products of TF32 round both factors, 2^-11 of each at most."""
    new = [70 if i % 170 == 3 else 1 for i in range(sequences)]
    p = D.Paged(new, [n + i % 50 for i, n in enumerate(new)], 1, 1, 64, 16, "float16", seed=80)
    w = torch.randn(64, 32, generator=torch.Generator().manual_seed(80))
    dev = G.attend_inputs(p)
    z = torch.empty(p.q.shape[0], 32, device="cuda")
    nodes = [("OxiPagedAttention", "attend", list(dev), ["out"], {"num_heads": 1, "kv_num_heads": 1}), ("MatMul", "product", ["out", "w"], ["z"], {})]
    s = G.session(nodes, dev, {"z": z}, {"w": w.numpy()})
    assert any(step["kernel"].startswith("umma") for step in s.steps()), s.steps()
    want, bound = D.attend(p)
    bound = bound @ w.double().abs() + (2 * 2.0**-11 + 66 * 2.0**-23) * (1 + 2.0**-10) * ((want.abs() + bound) @ w.double().abs())
    for _ in range(20):
        z.fill_(math.nan)
        G.run(s)
        G.within(z, want @ w.double(), bound)
