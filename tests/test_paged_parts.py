"""How many bf16 parts the probabilities of few queries take: attention emulated on the CPU, against the bound
that the GPU's outputs are held to (paged_cases.attention64 with HALF_16)."""
import pytest
import torch

from paged_cases import BF16, HALF_16, Batch, attention64, cancel_values, values64


def emulated(b, cache, q, scale, parts):
    """The last rows' outputs [sequences, heads, dim] with weights of so many bf16 parts, exact but for them
    and the output's rounding."""
    keys, values, ks, vs = cache
    G = q.shape[1] // b.hkv
    out = torch.zeros(len(b.lens), q.shape[1], b.dim)
    for i in range(len(b.lens)):
        p, o = b.places(i)
        K = values64(keys[p, :, o], None if ks is None else ks[p, :, o])
        for h in range(q.shape[1]):
            s = (K[:, h // G] @ q[int(b.off[i + 1]) - 1, h].double()) * scale
            w = torch.exp(s - s.max())
            total, weight = w.sum(), w if vs is None else w * vs[p, h // G, o].double()
            x, weight = weight, torch.zeros_like(weight)
            for _ in range(parts):
                weight += (x - weight).to(BF16).double()
            if vs is None:
                total = weight.sum()
            out[i, h] = ((weight @ values[p, h // G, o].double()) / total).to(BF16).float()
    return out


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q8", [False, True])
def test_parts_of_the_probabilities(dim, q8):
    b = Batch([1, 1, 2], [30, 200, 77], hkv=2, dim=dim, seed=61)
    cache, scale = b.cache(q8), 0.005
    q = b.randn(b.rows, 8, dim).to(BF16)
    cancel_values(b, cache, q, scale)
    want, bound = (t[(b.off[1:] - 1).long()] for t in attention64(b, *cache, q, scale, HALF_16))
    worst = [float(((emulated(b, cache, q, scale, n).double() - want).abs() / bound).max()) for n in (1, 2)]
    assert worst[0] > 2 and worst[1] < 1, worst
