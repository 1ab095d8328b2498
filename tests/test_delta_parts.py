"""How many bf16 parts the operands of the chunked delta rule need: its products emulated on the CPU, against
the limits that the GPU's states and outputs are held to (delta_cases.state_limit, output_limit)."""
import pytest
import torch

from delta_cases import (BF16, DeltaCase, concentrate_keys, final_states, output_error, output_limit, state_error,
                         state_limit)

CHUNK = 32


def parts(x, n):
    out = []
    for _ in range(n):
        out.append(x.to(BF16).float())
        x = x - out[-1]
    return out


def products(a, b, n):
    """a @ b of operands in n parts each, the products down to the size of the last part."""
    a, b = parts(a, n), parts(b, n)
    return sum(a[o - i] @ b[i] for o in reversed(range(n)) for i in range(o + 1))


def chunked(S, q, k, v, g, beta, scale, of_state, of_updates, of_outputs=2):
    """A head's outputs and final state [dv, dk] by chunks in float, its operands in so many bf16 parts."""
    out = []
    for a in range(0, len(k), CHUNK):
        qc, kc, vc, b = q[a:a + CHUNK], k[a:a + CHUNK], v[a:a + CHUNK], beta[a:a + CHUNK]
        G = g[a:a + CHUNK].double().cumsum(0)
        decay = torch.exp((G[:, None] - G[None]).clamp_max(0)).float()
        A = (b[:, None] * (kc @ kc.T) * decay).tril(-1)
        T = torch.linalg.solve_triangular(A + torch.eye(len(b)), torch.eye(len(b)), upper=False, unitriangular=True) * b
        P = sum(kc @ p.T for p in reversed(parts(S, of_state)))
        Y = vc - torch.exp(G).float()[:, None] * P
        U = products(T, Y, of_updates)
        M = ((qc @ kc.T) * decay).tril()
        seen = torch.exp(G).float()[:, None] * sum(qc @ p.T for p in reversed(parts(S, of_outputs)))
        out.append(((seen + products(M, U, of_outputs)) * scale).to(BF16))
        S = S * torch.exp(G[-1]).float()
        for p in reversed(parts(torch.exp(G[-1] - G).float()[:, None] * U, of_updates)):
            S = S + p.T @ kc
    return torch.cat(out), S


@pytest.mark.parametrize("decay", [0.0, 0.05])
def test_parts_of_the_operands(decay):
    c = DeltaCase([128, 70], 1, 2, 64, 64, seed=22, decay=decay)
    concentrate_keys(c)
    exact, want = final_states(c, torch.float64), c.exact()[0]
    q, k, v, g, beta = (t.float() for t in c.operands("cpu"))
    worst, outputs = {}, {}
    for of in ((3, 3), (2, 3), (3, 2), (3, 3, 1)):
        heads = [[chunked(c.states[int(c.origin[i])][h], q[a:b, 0], k[a:b, 0], v[a:b, h], g[a:b, h], beta[a:b, h],
                          c.scale, *of) for h in range(2)]
                 for i, (a, b) in enumerate(zip(c.off[:-1].tolist(), c.off[1:].tolist()))]
        states = torch.stack([torch.stack([S for _, S in seq]) for seq in heads])
        out = torch.cat([torch.stack([o for o, _ in seq], 1) for seq in heads])
        worst[of] = float((state_error(states, exact) / state_limit(c, exact)).max())
        outputs[of] = float((output_error(out, want) / output_limit(want)).max())
    assert outputs[3, 3] <= 1 and outputs[3, 3, 1] > 1.1, outputs
    assert worst[3, 3] <= 0.5          # what the kernels do
    assert worst[2, 3] > 1             # the state in two parts where its products come back into it
    assert worst[3, 2] > 4             # the updates in two
