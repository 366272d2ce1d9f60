"""The paged operators over many tokens, where sums grow long, work is shared among many and a lost token would hardly show:
equal values, planted keys, and errors held to what the roundings make on average."""
import numpy as np
import pytest
import torch

import emel_cpp_b200 as eb
from emel_cpp_b200 import paged
from tests import paged_plain as plain
from tests.test_gpu_paged import Cache, dev, done, filled, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = eb.Backend(0)
    yield b
    b.close()


def exact(q, k, v, scale, causal=True):
    """(result, root of the sum of (weight * value)^2) in 64 bits, a head at a time."""
    n, heads, _ = q.shape
    length, kv = k.shape[:2]
    out, root = (torch.empty(n, heads, v.shape[2], dtype=torch.float64, device=q.device) for _ in range(2))
    i, j = torch.arange(n, device=q.device)[:, None], torch.arange(length, device=q.device)[None]
    for h in range(heads):
        g = h // (heads // kv)
        s = q[:, h].double() @ k[:, g].double().T * scale
        if causal:
            s = s.masked_fill(j > length - n + i, -np.inf)
        p = torch.softmax(s, -1)
        out[:, h] = p @ v[:, g].double()
        root[:, h] = (p * p @ (v[:, g].double() ** 2)).sqrt()
    return out, root


def rms(x):
    return float(x.double().square().mean().sqrt())


def check_rms(got, want, root, weight_step, t, score=0.0):
    """Roundings of weights are independent of one another: together about weight_step * root; the result has one more.  Twice that, and
    what errors of the scores make (`score`, relative to root: they are independent, too)."""
    err, bound = rms(got.double() - want), 2 * ((weight_step + score) * rms(root) + plain.HALF_STEP[t] * rms(want))
    assert np.isfinite(err) and err <= bound, (err, bound)


# ---------------------------------------------------------------- packed prompts
@pytest.mark.parametrize("keys,dim,t,lift", [((1 << 20) + 3, 8, "f16", 0.5), (1 << 20, 128, "f16", 0.0), (1 << 22, 8, "bf16", 0.3), (1 << 25, 8, "f16", 0.5)])
def test_packed_equal_values_of_many_keys(be, keys, dim, t, lift):
    """All keys alike but the first, whose score is 2^lift above: sums of equal numbers, where every rounding goes the same way.  The
    tensor cores cut a sum's 17 addends (16 products, O) off at a unit of 2^-23 of O or less, O grows over 512 such products; a weight and a
    result have a rounding each, the sums f32 ones: of 64 weights, 64 tiles, the rest."""
    dt = plain.TORCH[t]
    q, k = torch.zeros(1, 1, dim, device="cuda", dtype=dt), torch.zeros(keys, 1, dim, device="cuda", dtype=dt)
    q[..., 0], k[0, 0, 0] = 1, lift
    v = torch.empty(keys, 1, dim, device="cuda", dtype=dt).copy_(torch.linspace(-3, 2, dim, device="cuda").to(dt))
    out, begin = torch.zeros_like(q), [dev([0, 1]), dev([0, keys])]
    torch.cuda.synchronize()
    done(be, be.attend_packed(paged.packed_request(q, k, v, out, t, *begin, 1, 1, 1, dim, 1, keys, causal=False, scale=float(np.log(2)))))
    want = v[0].double()
    rel = 2 * plain.HALF_STEP[t] + 256 * 17 * 2.0 ** -23 + (64 + 64 + keys / 8192) * 2.0 ** -24 + 2.0 ** -20
    assert ((out[0].double() - want).abs() <= rel * want.abs()).all(), float(((out[0].double() - want) / want).abs().max())


@pytest.mark.parametrize("queries,keys,heads,kv,dim,t,ramp", [
    (3, 30000, 4, 2, 128, "f16", 0.0), (200, 17000, 2, 1, 64, "bf16", 4.0), (300, 8192 + 128, 2, 2, 128, "f16", -4.0), (70, 8193, 8, 1, 40, "f16", 8.0),
    (5, 100003, 2, 2, 64, "bf16", 0.0), (129, 16384, 1, 1, 128, "bf16", 2.0),
])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_far_errors(be, queries, keys, heads, kv, dim, t, ramp, causal):
    """Random rows whose scores rise (ramp > 0), so that the running maximum moves all the way, or fall, or neither."""
    g, dt = gen(keys), plain.TORCH[t]
    q = torch.randn(queries, heads, dim, generator=g, device="cuda")
    k, v = (torch.randn(keys, kv, dim, generator=g, device="cuda") for _ in range(2))
    q[..., 0], k[..., 0] = 1.0, torch.linspace(0, ramp * dim ** 0.5, keys, device="cuda")[:, None]
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    out, begin = torch.full_like(q, 7.0), [dev([0, queries]), dev([0, keys])]
    torch.cuda.synchronize()
    req = paged.packed_request(q, k, v, out, t, *begin, 1, heads, kv, dim, queries, keys, causal=causal)
    done(be, be.attend_packed(req))
    want, root = exact(q, k, v, dim ** -0.5, causal)
    check_rms(out, want, root, plain.HALF_STEP[t], t)
    first = out.clone()
    done(be, be.attend_packed(req))
    assert torch.equal(first, out)


@pytest.mark.parametrize("keys,dim", [(20000, 64), (8200, 128)])
def test_packed_planted_keys(be, keys, dim):
    """One key takes all of a row's weight: at both sides of every kind of border (tiles of 128, moves of 64 tiles, the ends)."""
    g = gen(keys)
    at = sorted({p for b in (0, 128, 256, 1024, 4096, 8192, 16384, keys) for p in (b - 2, b - 1, b, b + 1) if 0 <= p < keys})
    k = torch.randn(keys, 1, dim, generator=g, device="cuda").sign().bfloat16()
    v = torch.randn(keys, 1, dim, generator=g, device="cuda").bfloat16()
    q = (k[at] * 16).contiguous()                               # 2 * dim^0.5 nats between equal signs and any other sum
    out, begin = torch.zeros_like(q), [dev([0, len(at)]), dev([0, keys])]
    torch.cuda.synchronize()
    done(be, be.attend_packed(paged.packed_request(q, k, v, out, "bf16", *begin, 1, 1, 1, dim, len(at), keys, causal=False)))
    assert torch.equal(out, v[at])
