"""OxiPagedAttention where softmax leaves little room: scores of any size.  Queries and keys have one lane that is not 0, so that
scores are exact and what is expected follows from them alone."""
import math

import pytest

import decoder_oracle as D
import test_gpu_decoder as G

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def one_lane(new, total, size, kind, seed, heads=1):
    """A batch of one sequence whose queries and keys are 0, and the slots of its tokens in order."""
    p = D.Paged([new], [total], heads, 1, size, 16, kind, seed=seed)
    slots = torch.tensor([int(p.table[0, j // 16]) * 16 + j % 16 for j in range(total)])
    p.kc.view(-1, 1, size)[slots] = 0
    p.q[:] = 0
    return p, slots


def attend(p, scale):
    dev, out = G.attend_inputs(p), torch.full(p.q.shape, math.nan, dtype=D.TYPES[p.kind], device="cuda")
    s = G.session([("OxiPagedAttention", "attend", list(dev), ["out"], {"num_heads": p.heads, "kv_num_heads": 1, "scale": scale})], dev, {"out": out})
    G.run(s)
    first = out.clone()
    G.run(s)
    assert torch.equal(torch.nan_to_num(first), torch.nan_to_num(out))
    return out.double().cpu()


# ---- scores far from 0 -----------------------------------------------------------------------------
@pytest.mark.parametrize("kind,query,key", [("float16", 4.0, 60.0), ("float16", 1000.0, 1000.0), ("float16", 60000.0, 30000.0), ("bfloat16", 2.0**20, 2.0**12), ("bfloat16", 2.0**50, 2.0**40),
                                            ("bfloat16", 2.0**-3, 2.0**100)])
@pytest.mark.parametrize("new,total,size", [(1, 700, 64), (2, 3000, 128), (1, 700, 256), (150, 700, 64), (200, 1500, 128)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("scale", [1.0, 0.3])
def test_attention_of_scores_of_any_size(kind, query, key, new, total, size, sign, scale):
    """Keys of 16-bit numbers from `key` down, the scores far apart: the two largest are equal and share everything, wherever they
    lie, so that the output is the mean of their values (probabilities of 1, products and sums of two numbers exact to 2^-22), but
    for scores near one another, whose probabilities follow from the differences.  All scores negative: the smallest sizes win."""
    p, slots = one_lane(new, total, size, kind, seed=95)
    g = torch.Generator().manual_seed(96)
    keys = (key * (0.25 + 0.5 * torch.rand(total, generator=g))).to(D.TYPES[kind]).double()
    low = total - new  # every row sees the tokens up to here
    keys[low // 3], keys[low // 2] = (key, key) if sign > 0 else (key * 0.125, key * 0.125)
    p.kc.view(-1, 1, size)[slots, 0, 3] = (sign * keys).to(D.TYPES[kind])
    p.q[:, 3] = query
    values = p.vc.view(-1, 1, size)[slots, 0].double()
    got = attend(p, scale)
    # the attribute is an f32 number
    scores = sign * float(torch.tensor(query, dtype=D.TYPES[kind])) * p.kc.view(-1, 1, size)[slots, 0, 3].double().abs() * float(torch.tensor(scale, dtype=torch.float32))
    for row in range(new):
        n = low + row + 1
        s = scores[:n] - scores[:n].max()
        prob = torch.exp(s) / torch.exp(s).sum()
        want = prob @ values[:n]
        mean = prob @ values[:n].abs()
        # differences of exact scores, scaled once: 2^-22 of each
        off = (prob * (s.abs() * 2.0**-21 + 2.0**-20)) @ values[:n].abs()
        low_bits = 2.0**-25 * values[:n].abs().sum(0) if kind == "float16" else 0.0
        bound = D.rounding(kind, want) + 2 * D.half_step(kind) * mean + 2 * off + (n + 16) * 2.0**-22 * mean + low_bits
        assert not torch.isnan(got[row]).any(), f"NaN in row {row}"
        assert ((got[row] - want).abs() <= bound).all(), (row, ((got[row] - want).abs() - bound).max())
