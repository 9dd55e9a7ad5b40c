"""GPU parity of the AdamW step with moments in 32 and in 8 bits, of the optimizer over it, and of their refusals.

Against float64 (tolerances set before the first run): a new moment is two products and a sum in float32, so 2^-22 of the
magnitudes that enter it; the parameter's change collects a quotient and two roots, 2^-20 of its own magnitude, then one
rounding of the parameter's type (u = 2^-24, 2^-11, 2^-8). The 8-bit codes are defined to the bit by float32 operations in a
fixed order, each rounded correctly; roots are numpy's, as torch's on the CPU are not always. Against float64 a code may differ where its unrounded value lies within
2^-10 of a half."""
import numpy as np
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

fa = sub("enhancers.fused_adamw")
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SHAPES = [(1,), (255,), (256,), (257,), (16, 64), (33, 77), (5000,), (3, 5, 7), (0,), (4096, 3), (20000,)]
HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def make(shapes, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    ps = [(torch.randn(s, generator=g) * 0.1).to(dtype) for s in shapes]
    gs = [(torch.randn(s, generator=g) * 10.0 ** -(i % 4)).to(dtype) for i, s in enumerate(shapes)]
    return ps, gs


def flat(ts):
    """Tensors as the flat blocks of the moments, in float32."""
    pad = lambda t: torch.nn.functional.pad(t.reshape(-1).float(), (0, -t.numel() % 256))      # noqa: E731
    return torch.cat([pad(t) for t in ts])


def root(x):
    return torch.from_numpy(np.sqrt(x.numpy()))


def encode_avg(m):
    m = m.view(-1, 256)
    s = m.abs().amax(1)
    q = torch.round(root(m.abs() / torch.where(s > 0, s, 1.0)[:, None]) * 127.0)
    return torch.where(m < 0, -q, q).to(torch.int8).view(-1), s


def encode_sq(v):
    u = root(v).view(-1, 256)
    s = u.amax(1)
    q = torch.round(root(u / torch.where(s > 0, s, 1.0)[:, None]) * 255.0)
    return torch.where(u > 0, q.clamp(min=1), q).to(torch.uint8).view(-1), s


def decode(state):
    cm = state[0].view(-1, 256).float() * (1.0 / 127.0)
    cv = state[1].view(-1, 256).float() * (1.0 / 255.0)
    u = cv * cv * state[3][:, None]
    return (cm * cm.abs() * state[2][:, None]).view(-1), (u * u).view(-1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_against_float64(native, dtype, bits):
    dtype = getattr(torch, dtype)
    ps, _ = make(SHAPES, dtype, 1)
    params = [p.cuda() for p in ps]
    state = fa.adamw_state(params, bits)
    b1, b2 = HYPER["betas"]
    for step in range(1, 5):
        grads = make(SHAPES, dtype, 10 + step)[1]
        p0, g0 = flat([p.cpu() for p in params]).double(), flat(grads).double()
        m0, v0 = (t.cpu().double() for t in state.values())
        codes = [t.cpu() for t in state] if bits == 8 else None
        fa.adamw_step(params, [g.cuda() for g in grads], state, step, **HYPER)
        m, v = b1 * m0 + (1 - b1) * g0, b2 * v0 + (1 - b2) * g0 * g0
        move = HYPER["lr"] / (1 - b1 ** step) * m / (torch.sqrt(v / (1 - b2 ** step)) + HYPER["eps"])
        want = p0 * (1 - HYPER["lr"] * HYPER["weight_decay"]) - move
        got = flat([p.cpu() for p in params]).double()
        # (a moment off by 2^-22 of what enters it moves m / sqrt(v) by that over sqrt(v))
        room = 2.0 ** -20 * (move.abs() + HYPER["lr"] / (1 - b1 ** step) * (m0.abs() + g0.abs())
                             / (torch.sqrt(v / (1 - b2 ** step)) + HYPER["eps"])) + 2.0 ** -23 * p0.abs()
        err = (got - want).abs()
        assert bool((err <= room + UNIT[dtype] * want.abs() + (2.0 ** -24 if dtype == torch.float16 else 0)).all())
        if bits == 32:
            gm, gv = state.values()
            assert bool(((gm.cpu().double() - m).abs() <= 2.0 ** -22 * (m0.abs() + g0.abs())).all())
            assert bool(((gv.cpu().double() - v).abs() <= 2.0 ** -22 * (v0 + g0 * g0)).all())
            continue
        # the codes: to the bit in float32, and the nearest code of the float64 moments
        mf, vf = decode(codes)
        gf = g0.float()
        em, ev = encode_avg(mf * b1 + gf * (1 - b1)), encode_sq(vf * b2 + gf * gf * (1 - b2))
        for k, t in enumerate((em[0], ev[0], em[1], ev[1])):
            assert torch.equal(state[k].cpu(), t), k
        gm, gv = decode([t.cpu() for t in state])
        assert torch.equal(state.values()[0].cpu(), gm) and torch.equal(state.values()[1].cpu(), gv)
        top = m.abs().view(-1, 256).amax(1).clamp(min=1e-300)[:, None]
        x = 127 * torch.sqrt(m.abs().view(-1, 256) / top)
        assert float((state[0].cpu().double().abs().view(-1, 256) - x).abs().max()) <= 0.5 + 2.0 ** -10


def test_small_moments_keep_a_code(native):
    # one large gradient and 255 tiny ones in a block: no second moment that is not zero rounds to zero
    g = torch.full((256,), 1e-6, device="cuda")
    g[0], g[1] = 1.0, 0.0
    p = torch.zeros(256, device="cuda")
    state = fa.adamw_state([p], 8)
    fa.adamw_step([p], [g], state, 1, lr=0.1, weight_decay=0.0)
    v = state.exp_avg_sq.cpu()
    assert int(v[0]) == 255 and int(v[1]) == 0 and bool((v[2:] >= 1).all())
    for step in range(2, 40):
        fa.adamw_step([p], [g], state, step, lr=0.1, weight_decay=0.0)
    assert bool(torch.isfinite(p).all()) and float(p.abs().max()) < 0.1 * 40 * 1.01 and float(p[1]) == 0.0


@pytest.mark.parametrize("size", [1e-22, 1e-18, 1e-13, 1e-6, 1e12])
def test_codes_at_the_ends_of_the_range(native, size):
    # second moments from subnormal to huge, where the quick way to a code does not hold: to the bit all the same
    g = torch.Generator().manual_seed(3)
    grad = torch.randn(4096, generator=g) * size * 10.0 ** torch.empty(4096).uniform_(-3, 0, generator=g)
    p = torch.zeros(4096, device="cuda")
    state = fa.adamw_state([p], 8)
    m, v = torch.zeros(4096), torch.zeros(4096)
    for step in range(1, 4):
        fa.adamw_step([p], [grad.cuda()], state, step, betas=(0.9, 0.99))
        em, ev = encode_avg(m * 0.9 + grad * (1 - 0.9)), encode_sq(v * 0.99 + grad * grad * (1 - 0.99))
        for k, t in enumerate((em[0], ev[0], em[1], ev[1])):
            assert torch.equal(state[k].cpu(), t), (step, k)
        m, v = decode([t.cpu() for t in state])
    assert bool(torch.isfinite(p).all())


def test_many_tensors_offsets_and_order(native):
    # more tensors than one launch takes, at every alignment of their type, give what one call each gives
    n = 230
    buf, gbuf = (torch.randn(n * 400, device="cuda").to(torch.bfloat16) for _ in range(2))
    sizes = [1 + (37 * i) % 399 for i in range(n)]
    cut = lambda b: [b[400 * i + i % 9:400 * i + i % 9 + s] if s + i % 9 <= 400 else b[400 * i:400 * i + s]   # noqa: E731
                     for i, s in enumerate(sizes)]
    params, grads = cut(buf), cut(gbuf)
    alone = [p.clone() for p in params]
    before = buf.clone()
    state = fa.adamw_state(params, 8)
    fa.adamw_step(params, grads, state, 1, **HYPER)
    for p, q, g in zip(params, alone, grads):
        fa.adamw_step([q], [g.clone()], fa.adamw_state([q], 8), 1, **HYPER)
        assert torch.equal(p, q)
    # nothing between the tensors was written
    mask = torch.ones_like(buf, dtype=torch.bool)
    for m in cut(mask):
        m.zero_()
    assert torch.equal(buf[mask], before[mask])


def test_not_finite_gradients_stay_in_their_block(native):
    p = torch.ones(1024, device="cuda")
    g = torch.full((1024,), 0.1, device="cuda")
    g[300], g[600] = float("nan"), float("inf")
    state = fa.adamw_state([p], 8)
    fa.adamw_step([p], [g], state, 1)
    m, v = state.values()
    for t in (m, v):
        assert bool(torch.isfinite(t[:256]).all()) and bool(torch.isfinite(t[768:]).all())
        assert bool(torch.isnan(t[256:768]).all())
    assert bool(torch.isfinite(p[:300]).all()) and bool(torch.isnan(p[300])) and bool(torch.isfinite(p[601:]).all())


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_trains_and_resumes(native, bits):
    torch.manual_seed(0)
    target = torch.randn(64, 96, device="cuda")

    def run(p, opt, steps):
        for _ in range(steps):
            opt.zero_grad()
            loss = ((p.float() - target) ** 2).mean()
            loss.backward()
            opt.step()
        return float(loss)
    p = torch.nn.Parameter(torch.zeros(64, 96, device="cuda", dtype=torch.bfloat16))
    opt = fa.AdamW([p], lr=0.05, weight_decay=0.0, bits=bits)
    first = run(p, opt, 1)
    run(p, opt, 60)
    saved, at = opt.state_dict(), p.detach().clone()
    saved = {"state": {k: {n: v.clone() if isinstance(v, torch.Tensor) else v for n, v in d.items()}
                       for k, d in saved["state"].items()}, "param_groups": saved["param_groups"]}
    last = run(p, opt, 20)
    assert last < first / 20
    q = torch.nn.Parameter(at)
    other = fa.AdamW([q], lr=0.05, weight_decay=0.0, bits=bits)
    other.load_state_dict(saved)
    run(q, other, 20)
    assert torch.equal(p, q)


def test_step_marks_saved_tensors_stale(native):
    p = torch.nn.Parameter(torch.randn(32, device="cuda"))
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    fa.AdamW([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(native):
    p, g = torch.zeros(300, device="cuda"), torch.ones(300, device="cuda")
    state = fa.adamw_state([p], 8)
    for bad in (dict(params=[p], grads=[]), dict(params=[p], grads=[g.half()]), dict(params=[p], grads=[g[:299]]),
                dict(params=[p], grads=[g.cpu()]), dict(params=[p.double()], grads=[g.double()]),
                dict(params=[torch.zeros(600, device="cuda")[::2]], grads=[g])):
        with pytest.raises(ValueError):
            fa.adamw_step(**bad, state=state, step=1)
    for bad in (dict(step=0), dict(step=1.5), dict(step=1, betas=(1.0, 0.9)), dict(step=1, eps=-1.0),
                dict(step=1, lr=float("nan"))):
        with pytest.raises(ValueError):
            fa.adamw_step([p], [g], state, **bad)
    with pytest.raises(sub("_native").NativeError, match="blocks"):
        fa.adamw_step([p, p], [g, g], state, 1)                     # the state of one tensor for two
    with pytest.raises(ValueError, match="belong together"):
        fa.adamw_step([p], [g], fa.AdamWState(state[0], state[1]), 1)
    with pytest.raises(ValueError):
        fa.adamw_state([p], 16)
    with pytest.raises(ValueError):
        fa.adamw_state([])
    q, r = torch.nn.Parameter(p.clone()), torch.nn.Parameter(p.clone())
    opt = fa.AdamW([q, r])
    opt.step()                                                      # no gradients: nothing happens
    q.grad = g.clone()
    with pytest.raises(ValueError, match="no gradient"):
        opt.step()
