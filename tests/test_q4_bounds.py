"""The tolerance that chunks over the 4-bit cache are tested with (`q4_bounds`): an answer with a mistake in it
lies outside, one with the kernel's roundings inside. Mistakes and roundings are made in the oracle."""
import numpy as np
import pytest
import torch

from oracle import q4 as O
from q4_bounds import bound, rounded, worst


def _attend(q, K, V, scale, G, late=0, weights=lambda p: p):
    """`O.attend` with the causal limit `late` tokens further back and a rounding of the weights."""
    nq, HQ, d = q.shape
    n = K.shape[0]
    out = np.zeros((nq, HQ, d))
    for h in range(HQ):
        s = q[:, h] @ K[:, h // G].T * scale
        s[np.arange(n)[None] > (n - nq + np.arange(nq) - late)[:, None]] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = weights(p) @ V[:, h // G] / p.sum(-1, keepdims=True)
    return out


def _case(d, g, n, nq, dtype):
    rng = np.random.default_rng(n + d)
    k, v = rng.standard_normal((n, 1, d)), rng.standard_normal((n, 1, d))
    k[:, :, :3] *= 6
    K, V = (O.values(*O.quantise(x, g)) for x in (k, v))
    q = rng.standard_normal((nq, 2, d)).astype(np.float16).astype(np.float64)
    eps = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    return q, K, V, eps


SHAPES = [(64, 32, 1000, 150, 0.125), (128, 128, 5000, 40, 0.08), (128, 64, 6000, 64, 0.05), (64, 64, 300, 130, 0.125)]


def _type(x, dtype):
    """A result in its type, as 64 bits."""
    return torch.from_numpy(x).to({"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]).double().numpy()


@pytest.mark.parametrize("d,g,n,nq,scale", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_the_kernels_roundings_lie_within(d, g, n, nq, scale, dtype):
    q, K, V, eps = _case(d, g, n, nq, dtype)
    want, tol = bound(q, K, V, scale, 2, eps, g, True)
    k = rounded(K) + (rounded(K - rounded(K)) if dtype == "fp16" else 0)
    got = _type(_attend(q, k, rounded(V), scale, 2, weights=lambda p: rounded(p * 256) / 256), dtype)
    assert worst(got, want, tol) <= 1
    got = _type(_attend(q, K, V, scale, 2), dtype)
    assert worst(got, *bound(q, K, V, scale, 2, eps, g, False)) <= 1


@pytest.mark.parametrize("d,g,n,nq,scale", SHAPES)
@pytest.mark.parametrize("mistake", ["tile lost", "stale values", "a panel's values zero", "own token hidden", "one token more"])
def test_mistakes_lie_outside(d, g, n, nq, scale, mistake):
    q, K, V, eps = _case(d, g, n, nq, "fp16")
    want, tol = bound(q, K, V, scale, 2, eps, g, True)
    V, late = rounded(V), 0
    if mistake == "tile lost":
        V = np.delete(V, np.s_[64:192], 0)
        K = np.delete(K, np.s_[64:192], 0)
    elif mistake == "stale values":
        V[128:256] = V[0:128]
    elif mistake == "a panel's values zero":
        V[n // 2 // 16 * 16:][:16] = 0
    else:
        late = 1 if mistake == "own token hidden" else -1
    got = _type(_attend(q, K, V, scale, 2, late), "fp16")
    assert worst(got, want, tol) > 1
