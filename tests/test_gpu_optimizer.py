"""AdamW on the GPU: captured steps of a part of the parameters, the root's last bit, gradients that are not finite."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_of_a_part(pkg, bits):
    """Parameters a and b have been stepped together; a step of a alone gives a its own count.  Captured, that would be
    copied from the common one at each replay and never go on: it is refused, and after one such eager step a captured
    one counts on as eager steps do."""
    gen = torch.Generator(device=DEV).manual_seed(bits)
    start, grad = (torch.randn(300, 40, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
    runs = []
    for captured in (False, True):
        a, b = (torch.nn.Parameter(start.clone()) for _ in range(2))
        opt = pkg.AdamW([a, b], lr=1e-2, state_bits=bits)
        a.grad, b.grad = grad.clone(), grad.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            opt.step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        b.grad = None
        if captured:
            counts = [opt.state[p]["step"] for p in (a, b)]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                with pytest.raises(RuntimeError, match="eager"):
                    opt.step()
                start.clone()                               # a capture of nothing else would warn
            assert all(opt.state[p]["step"] is c for p, c in zip((a, b), counts))
            assert [int(c) for c in counts] == [1, 1]
            del graph
        opt.step()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        seen = []
        for rep in range(3):
            graph.replay() if captured else opt.step()
            torch.cuda.synchronize()
            s = opt.state[a]
            second = "exp_avg_sq" if bits == 32 else "exp_avg_sq_root"
            seen.append([t.clone() for t in (a.detach(), s["master"], s["exp_avg"].float(), s[second].float(), s["step"])])
            (start * 2).sum().item()                        # eager work between the replays
        assert [int(s[-1]) for s in seen] == [3, 4, 5] and int(opt.state[b]["step"]) == 1
        runs.append(seen)
    for x, y in zip(*runs):
        assert all(torch.equal(s, t) for s, t in zip(x, y))


def test_root_is_rounded_correctly(pkg):
    """m = 1, v given, no decay, p = 0, lr = 1, eps = 0 and corrections of 1 (1 - 2^-201): p = -1 / sqrt(v), the root
    and the quotient each rounded to nearest, as numpy rounds them."""
    n = 1 << 20
    rng = np.random.default_rng(7)
    v = np.exp2(rng.uniform(-120.0, 120.0, n)).astype(np.float32)
    v[:64] = np.float32(2.0) ** -149 * np.arange(1, 65, dtype=np.float32)          # subnormal numbers
    want = -(np.float32(1.0) / np.sqrt(v))
    p, g, m = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), torch.full((n,), 2.0, device=DEV)
    vt = torch.from_numpy(v * np.float32(2.0)).to(DEV)
    pkg.adamw_step([p], [g], [m], [vt], torch.full((1,), 200, dtype=torch.int64, device=DEV), lr=1.0, betas=(0.5, 0.5),
                   eps=0.0, weight_decay=0.0)
    assert (m == 1).all() and np.array_equal(vt.cpu().numpy(), v)
    wrong = int((p.cpu().numpy() != want).sum())
    assert wrong == 0, f"{wrong} of {n}"


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("bits", [32, 8])
def test_gradient_that_is_not_finite(pkg, bits, bad):
    """fp32 moments lose the element's own; in 8 bits its block of 128 becomes NaN, and the parameters one step later."""
    n = 300
    g = torch.full((n,), 0.5, device=DEV)
    p = torch.nn.Parameter(torch.ones(n, device=DEV))
    opt = pkg.AdamW([p], lr=1e-2, state_bits=bits)
    g[133] = bad
    hit, block = torch.zeros(n, dtype=torch.bool, device=DEV), torch.zeros(n, dtype=torch.bool, device=DEV)
    hit[133], block[128:256] = True, True
    p.grad = g
    opt.step()
    assert torch.equal(~torch.isfinite(p), hit)
    m = opt.state[p]["exp_avg"].float()
    assert torch.equal(~torch.isfinite(m), block if bits == 8 else hit)
    p.grad = torch.full((n,), 0.5, device=DEV)
    opt.step()
    assert torch.equal(~torch.isfinite(p), block if bits == 8 else hit)
