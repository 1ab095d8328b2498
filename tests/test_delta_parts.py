"""How many bf16 parts the operands of the chunked delta rule need: its products emulated on the CPU, against
the limit that the GPU's states are held to (delta_cases.state_limit)."""
import pytest
import torch

from delta_cases import BF16, DeltaCase, concentrate_keys, final_states, state_error, state_limit

CHUNK = 32


def parts(x, n):
    out = []
    for _ in range(n):
        out.append(x.to(BF16).float())
        x = x - out[-1]
    return out


def chunked(S, k, v, g, beta, of_state, of_updates):
    """A head's final state [dv, dk] by chunks in float, its operands in so many bf16 parts."""
    for a in range(0, len(k), CHUNK):
        kc, vc, b = k[a:a + CHUNK], v[a:a + CHUNK], beta[a:a + CHUNK]
        G = g[a:a + CHUNK].double().cumsum(0)
        decay = torch.exp((G[:, None] - G[None]).clamp_max(0)).float()
        A = (b[:, None] * (kc @ kc.T) * decay).tril(-1)
        T = torch.linalg.solve_triangular(A + torch.eye(len(b)), torch.eye(len(b)), upper=False, unitriangular=True) * b
        P = sum(kc @ p.T for p in reversed(parts(S, of_state)))
        Y = vc - torch.exp(G).float()[:, None] * P
        t, y = parts(T, of_updates), parts(Y, of_updates)
        U = sum(t[n - i] @ y[i] for n in reversed(range(of_updates)) for i in range(n + 1))
        S = S * torch.exp(G[-1]).float()
        for p in reversed(parts(torch.exp(G[-1] - G).float()[:, None] * U, of_updates)):
            S = S + p.T @ kc
    return S


@pytest.mark.parametrize("decay", [0.0, 0.05])
def test_parts_of_the_operands(decay):
    c = DeltaCase([128, 70], 1, 2, 64, 64, seed=22, decay=decay)
    concentrate_keys(c)
    exact = final_states(c, torch.float64)
    _, k, v, g, beta = (t.float() for t in c.operands("cpu"))
    worst = {}
    for of in ((3, 3), (2, 3), (3, 2)):
        states = torch.stack([torch.stack([
            chunked(c.states[int(c.origin[i])][h], k[a:b, 0], v[a:b, h], g[a:b, h], beta[a:b, h], *of) for h in range(2)])
            for i, (a, b) in enumerate(zip(c.off[:-1].tolist(), c.off[1:].tolist()))])
        worst[of] = float((state_error(states, exact) / state_limit(c, exact)).max())
    assert worst[3, 3] <= 0.5          # what the kernels do
    assert worst[2, 3] > 1             # the state in two parts where its products come back into it
    assert worst[3, 2] > 4             # the updates in two
