"""AdamW on the GPU: captured steps of a part of the parameters, the root's last bit, gradients that are not finite, long
lists in 8 bits, the size and sign of a first update."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_adamw import BETAS, DECAY, EPS, LR, exponents, mix, pack, tensors  # noqa: E402

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


def test_many_tensors_in_8_bits(pkg):
    """130 tensors, three launches: parameters, masters and m's codes as each by itself (they do not go by the place in
    the list), the root's codes by the dither of the place."""
    shapes = [(1 + 37 * k % 700,) for k in range(130)]
    s = tensors(torch.bfloat16, 8, True, 3, shapes)
    pack(pkg, s)
    buf = torch.empty(s["params"][5].numel() + 1, dtype=torch.bfloat16, device=DEV)       # an odd address
    buf[1:].copy_(s["params"][5])
    s["params"][5] = buf[1:]
    wide = torch.empty(s["grads"][6].numel(), 2, dtype=torch.bfloat16, device=DEV)        # a strided gradient
    wide[:, 0] = s["grads"][6]
    s["grads"][6] = wide[:, 0]

    def copy(x):
        return tuple(t.clone() for t in x) if isinstance(x, tuple) else x.clone()
    alone = {k: [copy(x) for x in v] for k, v in s.items()}
    r0 = [pkg.unpack_moment(x).cpu().numpy() for x in s["v"]]
    seed, kw = 4, dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY)
    pkg.adamw_step(s["params"], s["grads"], s["m"], s["v"], torch.zeros(1, dtype=torch.int64, device=DEV),
                   masters=s["masters"], seed=seed, **kw)
    f = np.float32
    b2, ob2 = f(BETAS[1]), f(1 - BETAS[1])
    for i in range(len(shapes)):
        one = {k: [v[i]] for k, v in alone.items()}
        pkg.adamw_step(one["params"], one["grads"], one["m"], one["v"], torch.zeros(1, dtype=torch.int64, device=DEV),
                       masters=one["masters"], seed=seed, **kw)
        assert torch.equal(one["params"][0], s["params"][i]) and torch.equal(one["masters"][0], s["masters"][i]), i
        for a, b in zip(one["m"][0], s["m"][i]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i
        # the root in numpy's fp32, operation by operation
        g = alone["grads"][i].float().cpu().numpy()
        n = g.size
        r = np.sqrt((r0[i] * r0[i]) * b2 + (g * g) * ob2)
        e = exponents(np.concatenate([r, np.zeros(-n % 128, dtype=np.float32)]))
        a = r.astype(np.float64) / np.repeat(np.exp2(e.astype(np.float64)), 128)[:n]
        h = mix(np.arange((n + 1) // 2, dtype=np.uint64) * np.uint64(0x9E3779B9)
                + mix(np.uint64((seed + 0x9E3779B9 + i * 0xBB67AE85) & 0xFFFFFFFF)))
        u = np.stack([h & np.uint64(0xFFFF), h >> np.uint64(16)], -1).reshape(-1)[:n].astype(np.float64) / 65536
        q = np.exp2(np.maximum(np.frexp(a)[1] - 1, -6).astype(np.float64) - 3)
        k = np.floor((a / q).astype(np.float32) + u.astype(np.float32))
        k = np.where((a > 0) & (k < 1), 1, k)
        codes, scales = s["v"][i]
        assert np.array_equal(scales.cpu().numpy().astype(int) - 127, e), i
        assert np.array_equal(codes.cpu().float().numpy().astype(np.float64), k * q), i


@pytest.mark.parametrize("bits", [32, 8])
def test_first_update(pkg, bits):
    """Without decay the first update is lr g / (|g| + eps): its size and sign, for every element of a training step's
    parameters (FP8 linears, a modulated norm), in the master weights."""
    torch.manual_seed(3)
    D, F, lr = 256, 640, 1e-3
    up, down = (pkg.make_linear("fp8", i, o, device=DEV, dtype=torch.bfloat16) for i, o in ((D, F), (F, D)))
    e = torch.nn.Parameter((torch.randn(1, 6, D, device=DEV) * 0.1).to(torch.bfloat16))
    params = [e, *up.parameters(), *down.parameters()]
    opt = pkg.AdamW(params, lr=lr, weight_decay=0.0, state_bits=bits)
    x = torch.randn(2, 300, D, device=DEV).to(torch.bfloat16)
    h = pkg.modulated_layer_norm(x, e.chunk(6, dim=1)[3], e.chunk(6, dim=1)[4])
    (x + down(torch.nn.functional.gelu(up(h), approximate="tanh"))).float().square().mean().backward()
    before = [p.detach().float() for p in params]
    opt.step()
    u = 2.0 ** -24
    for p, b in zip(params, before):
        g = p.grad.double()
        want = lr * g / (g.abs() + 1e-8)
        moved = b.double() - opt.state[p]["master"].double()
        # m and v are (1 - b) g and (1 - b) g^2, the corrections undo it: 16 roundings of the quotient; the difference
        # from the parameter one more of its value.  (1 - b2 as a float is off by half a step, its root by a quarter.)
        # A gradient below 1e-19 would lose its square.
        big = g.abs() > 1e-19
        assert ((moved - want).abs() <= 16 * u * want.abs() + u * (b.double().abs() + lr))[big].all()
        assert big.any() and (moved * g >= 0).all()
        assert torch.equal(p.detach(), opt.state[p]["master"].to(torch.bfloat16))
