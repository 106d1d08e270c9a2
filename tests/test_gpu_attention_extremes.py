"""OxiPagedAttention where softmax leaves little room: scores of any size, and long tails of small probabilities.  Queries and keys
have one lane that is not 0, so that scores are exact and what is expected follows from them alone."""
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


# ---- long tails of small probabilities -----------------------------------------------------------
@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("new,total,size", [(1, 40000, 64), (1, 3000, 128), (1, 3000, 256), (3, 40000, 64), (80, 40000, 64), (70, 6000, 128)])
@pytest.mark.parametrize("gap", [11.0, 17.6, 19.5])
def test_attention_keeps_what_many_small_probabilities_sum_up_to(new, total, size, gap, kind):
    """One key takes nearly everything, in a value of 0; the others' exponentials, exp(-gap) each, are all that the output is
    made of.  Each is rounded to the 16-bit type: half a step, and of f16 below its least normal number 2^-25 of what one is
    written as.  The kernels write 2^15 (streamed) and 2^11 (tiles) for the largest, so that e^-19.5 = 2^-28.1 loses 2^-36 at
    most, 0.4 % of it; the f32 sums lose (t + 16) * 2^-22."""
    p = D.Paged([new], [total], 1, 1, size, 16, kind, seed=91)
    flat = lambda c: c.view(-1, 1, size)  # noqa: E731
    slots = torch.tensor([int(p.table[0, j // 16]) * 16 + j % 16 for j in range(total)])
    flat(p.kc)[slots] = 0
    flat(p.vc)[slots] = 1
    at = slots[total // 2]
    flat(p.kc)[at, 0, 0] = gap / 4  # a 16-bit number: the definition takes it as it is
    flat(p.vc)[at] = 0
    p.q[:] = 0
    p.q[:, 0] = 4
    s, dev, out = G.check_attend(p, scale=1.0)
    score = 4 * float(p.kc.view(-1, 1, size)[at, 0, 0])
    for i in range(new):
        others = total - new + i
        tail = others * math.exp(-score)
        want = torch.full((size,), tail / (1 + tail), dtype=torch.float64)
        off = 2 * D.half_step(kind) + (2.0**-36 / math.exp(-score) if kind == "float16" else 0) + (total + 16) * 2.0**-22 + 2 * (size + 4) * 2.0**-23 * score
        G.within(out[i], want, D.rounding(kind, want) + off * want)
