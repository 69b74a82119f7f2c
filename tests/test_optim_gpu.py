"""The AdamW step over many tensors (ops.adamw_step, ops.grad_norm, optim.AdamW) on the GPU against the step in 64 bits, and the
8-bit moments bit for bit against elementary float32 operations."""
import numpy as np
import pytest
import torch

from tests import adamw_oracle as A

pytestmark = pytest.mark.gpu
DEV = 'cuda'
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def _grads(shape, rng, dtype=torch.float32):
    size = np.exp(1.5 * rng.standard_normal((shape[0],) + (1,) * (len(shape) - 1)) - 4) if shape else 0.1
    return torch.from_numpy(np.asarray(size * rng.standard_normal(shape), dtype=np.float32)).to(DEV).to(dtype)


def _params(shape, rng, dtype=torch.float32):
    return torch.from_numpy(np.asarray(0.1 * rng.standard_normal(shape), dtype=np.float32)).to(DEV).to(dtype)


def _zeros8(p):
    n = -(-p.numel() // 128)
    return (torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e5m2),
            torch.zeros(n, 2, device=DEV))


def _flat(t):
    """numpy values of t in memory order (uint8 for 8-bit codes, float64 else)."""
    t = t.detach()
    if t.dtype in (torch.float8_e4m3fn, torch.float8_e5m2):
        t = t.view(torch.uint8)
    if t.dim() and not t.is_contiguous():
        order = sorted(range(t.dim()), key=lambda d: -t.stride(d))
        t = t.permute(order)
    a = t.cpu()
    return (a.numpy() if a.dtype == torch.uint8 else a.double().numpy()).reshape(-1)


def _check32(p0, g, m0, v0, t, p1, m1, v1, factor=1.0, hyper=HYPER):
    e = A.step64(_flat(p0), _flat(g), _flat(m0), _flat(v0), t, hyper['lr'], *hyper['betas'], hyper['eps'], hyper['weight_decay'], factor)
    half = HALF_STEP[p1.dtype]
    tiny = 2.0 ** -25 if p1.dtype == torch.float16 else 0.                       # half of fp16's smallest step
    assert (np.abs(_flat(p1) - e[0]) <= e[3] + half * (np.abs(e[0]) + e[3]) + tiny).all()
    assert (np.abs(_flat(m1) - e[1]) <= e[4]).all() and (np.abs(_flat(v1) - e[2]) <= e[5]).all()


SHAPES = [[(1,)], [(7,), (8,), (9,)], [(127,), (128, 1), (3, 43)], [(2047,), (2048,), (2049,), (5, 1000)], [(), (0, 4), (300, 64), (1,)]]


@pytest.mark.parametrize('dtype,grad_dtype', [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                              (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize('shapes', range(len(SHAPES)))
def test_float32_moments_follow_the_step_in_64_bits(shapes, dtype, grad_dtype):
    from igcn_cf_amd import ops
    rng = np.random.default_rng(shapes)
    ps = [_params(s, rng, dtype) for s in SHAPES[shapes]]
    ms, vs = [torch.zeros_like(p, dtype=torch.float32) for p in ps], [torch.zeros_like(p, dtype=torch.float32) for p in ps]
    ts = [torch.full((), float(i), device=DEV) for i in range(len(ps))]            # every tensor counts its own steps
    for step in range(1, 4):
        gs = [_grads(s, rng, grad_dtype) for s in SHAPES[shapes]]
        before = [(p.clone(), m.clone(), v.clone()) for p, m, v in zip(ps, ms, vs)]
        assert ops.adamw_step(ps, gs, ms, vs, ts, **HYPER) is None
        for i, (p0, m0, v0) in enumerate(before):
            assert float(ts[i]) == i + step
            _check32(p0, gs[i], m0, v0, i + step, ps[i], ms[i], vs[i])


@pytest.mark.parametrize('shapes', range(len(SHAPES)))
@pytest.mark.parametrize('dtype,clip', [(torch.float32, False), (torch.float32, True), (torch.bfloat16, True), (torch.float16, False)])
def test_8_bit_moments_meet_the_elementary_operations_bit_for_bit(shapes, dtype, clip):
    from igcn_cf_amd import ops
    rng = np.random.default_rng(100 + shapes)
    seed = 0x1234567890abcdef
    ps = [_params(s, rng, dtype) for s in SHAPES[shapes]]
    state = [_zeros8(p) for p in ps]
    ts = [torch.zeros((), device=DEV) for _ in ps]
    b1, b2 = HYPER['betas']
    for step in range(1, 5):
        gs = [_grads(s, rng, dtype) for s in SHAPES[shapes]]
        before = [(p.clone(), _flat(m), _flat(v), s.cpu().numpy()) for p, (m, v, s) in zip(ps, state)]
        norm = ops.adamw_step(ps, gs, [s[0] for s in state], [s[1] for s in state], ts, scales=[s[2] for s in state], seed=seed,
                              max_grad_norm=0.05 if clip else None, **HYPER)
        factor = np.float32(min(1.0, 0.05 / (float(np.sqrt(sum((_flat(g) ** 2).sum() for g in gs))) + 1e-6))) if clip else np.float32(1)
        assert (norm is not None) == clip
        for i, (p0, mc0, vc0, s0) in enumerate(before):
            mc, vc, sc, m, v = A.moments8(_flat(gs[i]).astype(np.float32), mc0, vc0, s0, factor, b1, b2, seed, i, step)
            assert np.array_equal(_flat(state[i][0]), mc) and np.array_equal(_flat(state[i][1]), vc)
            assert np.array_equal(state[i][2].cpu().numpy(), sc)
            m0, v0 = (A.decode(c, k, b).astype(np.float64) * np.repeat(s0[:, j], 128)[:c.size] for j, (c, k, b) in enumerate(((mc0, 3, 7), (vc0, 2, 15))))
            e = A.step64(_flat(p0), _flat(gs[i]), m0, v0, step, HYPER['lr'], b1, b2, HYPER['eps'], HYPER['weight_decay'], float(factor))
            assert (np.abs(_flat(ps[i]) - e[0]) <= e[3] + HALF_STEP[dtype] * (np.abs(e[0]) + e[3]) + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
            # what is held is within one code step of the average: 1/8 of its size (e4m3), 1/4 (e5m2), or the smallest step of the block
            held_m = A.decode(mc, 3, 7).astype(np.float64) * np.repeat(sc[:, 0], 128)[:mc.size]
            held_v = A.decode(vc, 2, 15).astype(np.float64) * np.repeat(sc[:, 1], 128)[:vc.size]
            assert (np.abs(held_m - m) <= np.abs(m) / 8 * (1 + 1e-6) + np.repeat(sc[:, 0], 128)[:mc.size] * 2.0 ** -9).all()
            assert (np.abs(held_v - v) <= v / 4 * (1 + 1e-6) + np.repeat(sc[:, 1], 128)[:vc.size] * 2.0 ** -16).all()
            assert ((vc > 0) == (v * np.repeat(sc[:, 1] > 0, 128)[:v.size] > 0)).all()


def test_torch_reads_the_codes_as_the_moments_they_stand_for():
    from igcn_cf_amd import ops
    rng = np.random.default_rng(5)
    p, g = _params((33, 40), rng), _grads((33, 40), rng)
    m8, v8, s = _zeros8(p)
    ops.adamw_step([p], [g], [m8], [v8], [torch.zeros((), device=DEV)], scales=[s], **HYPER)
    for t, k, b in ((m8, 3, 7), (v8, 2, 15)):
        assert np.array_equal(t.float().cpu().numpy().reshape(-1), A.decode(t.view(torch.uint8).cpu().numpy().reshape(-1), k, b))


def test_stochastic_rounding_is_right_in_the_mean_and_does_not_freeze_the_average():
    """4 096 seeds round the same averages: the mean of what is held is off by at most 6 standard deviations of such a mean (a rounding
    to one of two neighbours a step apart varies by at most half a step).  And a second moment that has to rise a thousandfold at 0.1 %
    of its target a step gets there: rounded to nearest, a step under an eighth of its size would leave it where it was."""
    from igcn_cf_amd import ops
    rng = np.random.default_rng(6)
    g = _grads((128,), rng)
    mean = [0., 0.]
    n = 4096
    for seed in range(n):
        p = torch.zeros(128, device=DEV)
        m8, v8, s = _zeros8(p)
        ops.adamw_step([p], [g], [m8], [v8], [torch.zeros((), device=DEV)], scales=[s], seed=seed * 0x9e3779b97f4a7c15, **HYPER)
        mean[0] = mean[0] + m8.double() * s[0, 0].double() / n
        mean[1] = mean[1] + v8.double() * s[0, 1].double() / n
    true = (0.1 * g.double(), 0.001 * g.double() ** 2)
    for got, want, part, scale, small in zip(mean, true, (8, 4), s[0].double(), (2.0 ** -9, 2.0 ** -16)):
        step = torch.maximum(want.abs() / part, scale * small)
        some = want.abs() > 2 * scale * small                                        # (a second moment under the smallest code is held as that code)
        assert bool(((got - want).abs() <= 6 * step / 2 / n ** 0.5 + 1e-6 * want.abs())[some].all())
    p = torch.zeros(256, device=DEV)
    m8, v8, s = _zeros8(p)
    t = torch.zeros((), device=DEV)
    small, large = torch.full((256,), 1e-3, device=DEV), torch.full((256,), 1e-3, device=DEV)
    small[::128] = large[::128] = 1e-1                                               # one large value in each block sets its scale
    large[1::2] = 3e-2
    for k in range(6000):
        ops.adamw_step([p], [small if k < 1000 else large], [m8], [v8], [t], scales=[s], lr=0.)
    v = (v8.float() * s[:, 1].repeat_interleave(128)).double()
    want = 9e-4 * (1 - 0.999 ** 5000)
    # a step moves v by at most 0.1 %, so it lands on the next code (a quarter off at most) with a chance of 0.001 / 0.25 at least: a walk of
    # variance 0.001 * 0.25 a step, pulled back over 1 000 steps: 0.125, 35 % of v; the mean of 128 such values is within 0.16 (5 sigma)
    assert abs(float(v[1::2].mean()) / want - 1) < 0.16 and float(v[1::2].min()) > want / 4


@pytest.mark.parametrize('eight', [False, True])
def test_orders_offsets_and_many_tensors(eight):
    """Transposed parameters (dense, not contiguous), views that start off any alignment, and more tensors than one launch takes give
    what contiguous, aligned, single calls give."""
    from igcn_cf_amd import ops
    rng = np.random.default_rng(7)
    shapes = [((i * 37) % 311 + 1, i % 5 + 1) for i in range(130)]
    base = [_params((s[0] * s[1] + 3,), rng) for s in shapes]
    gbase = [_grads((s[0] * s[1] + 3,), rng) for s in shapes]
    view = [(lambda b, s, o, tr: b[o:o + s[0] * s[1]].view(s[::-1]).t() if tr else b[o:o + s[0] * s[1]].view(s)) for _ in shapes]
    ps = [f(b, s, i % 4 and 1, i % 3 == 0) for i, (f, b, s) in enumerate(zip(view, [b.clone() for b in base], shapes))]
    gs = [f(b, s, (i + 1) % 3, i % 3 == 0) for i, (f, b, s) in enumerate(zip(view, gbase, shapes))]
    if eight:
        st = [_zeros8(p) for p in ps]
        ms, vs, sc = [s[0] for s in st], [s[1] for s in st], [s[2] for s in st]
    else:
        ms, vs, sc = [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps], None
    ts = [torch.zeros(1, device=DEV) for _ in ps]
    p0 = [p.clone() for p in ps]
    norm = ops.adamw_step(ps, gs, ms, vs, ts, scales=sc, max_grad_norm=0.5, seed=3, **HYPER)
    factor = min(1.0, 0.5 / (float(np.sqrt(sum((_flat(g) ** 2).sum() for g in gs))) + 1e-6))
    assert abs(float(norm) - float(np.sqrt(sum((_flat(g) ** 2).sum() for g in gs)))) <= 2.0 ** -23 * float(norm)
    for i in range(len(ps)):
        n = ps[i].numel()
        e = A.step64(_flat(p0[i]), _flat(gs[i]), np.zeros(n), np.zeros(n), 1, HYPER['lr'], *HYPER['betas'], HYPER['eps'], HYPER['weight_decay'], factor)
        assert (np.abs(_flat(ps[i]) - e[0]) <= e[3] + 2.0 ** -24 * np.abs(e[0])).all(), i
        if eight:
            mc, vc, s, _, _ = A.moments8(_flat(gs[i]).astype(np.float32), np.zeros(n, np.uint8), np.zeros(n, np.uint8), np.zeros((-(-n // 128), 2), np.float32),
                                         np.float32(factor), 0.9, 0.999, 3, i, 1)
            assert np.array_equal(_flat(ms[i]), mc) and np.array_equal(_flat(vs[i]), vc) and np.array_equal(sc[i].cpu().numpy(), s), i
        else:
            assert (np.abs(_flat(ms[i]) - e[1]) <= e[4]).all() and (np.abs(_flat(vs[i]) - e[2]) <= e[5]).all(), i
    for i, b in enumerate(base):                                                     # nothing outside a view is touched
        whole = ps[i]._base if ps[i]._base is not None else ps[i]
        o, n = i % 4 and 1, ps[i].numel()
        assert torch.equal(whole[:o], b[:o]) and torch.equal(whole[o + n:], b[o + n:])


def test_norm_over_many_tensors_and_clipping_by_a_given_one():
    from igcn_cf_amd import ops
    rng = np.random.default_rng(8)
    for dtypes in ((torch.float32,), (torch.float32, torch.bfloat16, torch.float16)):
        gs = [_grads(s, rng, dtypes[i % len(dtypes)]) for i, s in enumerate([(1,), (0, 3), (1000003,), (64, 129), ()] * 30)]
        want = float(np.sqrt(sum((_flat(g) ** 2).sum() for g in gs)))
        got = ops.grad_norm(gs)
        assert got.dtype == torch.float32 and got.dim() == 0 and abs(float(got) - want) <= 2.0 ** -23 * want
        assert torch.equal(ops.grad_norm(gs), got)                                   # same order every time
    assert float(ops.grad_norm([])) == 0. and float(ops.grad_norm([torch.empty(0, device=DEV)])) == 0.
    assert not np.isfinite(float(ops.grad_norm([torch.tensor([1., float('nan')], device=DEV)])))
    p0, g = _params((5, 77), rng), _grads((5, 77), rng)
    out = []
    for norm in (None, torch.full((), 4.0, device=DEV)):
        p, m, v = p0.clone(), torch.zeros_like(p0), torch.zeros_like(p0)
        got = ops.adamw_step([p], [g], [m], [v], [torch.zeros((), device=DEV)], max_grad_norm=1e-3, grad_norm=norm, **HYPER)
        assert norm is None or got is norm
        _check32(p0, g, torch.zeros_like(p0), torch.zeros_like(p0), 1, p, m, v, factor=1e-3 / (float(got) + 1e-6))
        out.append(m)
    assert not torch.equal(*out)


@pytest.mark.parametrize('eight', [False, True])
def test_zero_huge_and_broken_gradients(eight):
    """All-zero gradients from zero moments move nothing but the decay; a NaN or an infinity shows in its own parameter at once and, with
    8-bit moments, as a NaN scale of its block — never in another block; gradients whose squares leave the codes' range are held as zero."""
    from igcn_cf_amd import ops
    for case in ('zero', 'tiny', 'nan', 'inf'):
        p0 = torch.linspace(-1, 1, 400, device=DEV)
        g = torch.zeros(400, device=DEV)
        if case == 'tiny':
            g.fill_(1e-20)
        elif case != 'zero':
            g.fill_(0.01)
            g[130] = float(case)
        p = p0.clone()
        m, v, s = _zeros8(p) if eight else (torch.zeros_like(p), torch.zeros_like(p), None)
        ops.adamw_step([p], [g], [m], [v], [torch.zeros((), device=DEV)], scales=[s] if eight else None, **HYPER)
        if case in ('zero', 'tiny'):
            keep = p0.double() * (1 - HYPER['lr'] * HYPER['weight_decay'])
            assert bool(((p.double() - keep).abs() <= 4 * 2.0 ** -24 * p0.abs().double() + 1e-13).all())        # (1e-20 / eps * lr / 0.1)
            if eight:
                assert not v.view(torch.uint8).any() and bool((s[:, 1] == 0).all())
                assert case == 'tiny' or not s.any()
        else:
            broken = ~torch.isfinite(p)
            assert broken.nonzero().flatten().tolist() == [130]
            if eight:
                assert torch.isnan(s).all(1).tolist() == [False, True, False, False] and not m.view(torch.uint8)[128:256].any()


def test_captured_steps_follow_the_eager_ones():
    """A captured step (clipped, 8-bit and float32 moments, a device learning rate) replayed with the program's own work between replays
    gives what eager calls give, bit for bit; its steps go on counting."""
    from igcn_cf_amd import ops
    rng = np.random.default_rng(9)
    p0 = [_params((300, 64), rng), _params((1000,), rng)]
    grads = [[_grads((300, 64), rng), _grads((1000,), rng)] for _ in range(6)]
    for eight in (False, True):
        ends = []
        for captured in (False, True):
            ps = [p.clone() for p in p0]
            st = [_zeros8(p) if eight else (torch.zeros_like(p), torch.zeros_like(p), None) for p in ps]
            ts, lr = [torch.zeros((), device=DEV) for _ in ps], torch.full((1,), 1e-2, device=DEV)
            gs = [g.clone() for g in grads[0]]
            run = lambda: ops.adamw_step(ps, gs, [s[0] for s in st], [s[1] for s in st], ts, lr=lr, weight_decay=0.01, max_grad_norm=0.1,
                                         scales=[s[2] for s in st] if eight else None, seed=11)
            if captured:
                saved = [[t.clone() for t in (*ps, *ts, *(x for s in st for x in s if x is not None))]]
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    run()
                torch.cuda.current_stream().wait_stream(side)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    norm = run()
                for t, o in zip((*ps, *ts, *(x for s in st for x in s if x is not None)), saved[0]):
                    t.copy_(o)
            norms = []
            for k in range(6):
                for a, b in zip(gs, grads[k]):
                    a.copy_(b)
                lr.fill_(1e-2 / (k + 1))
                if captured:
                    graph.replay()
                else:
                    norm = run()
                norms.append(float(norm))
                junk = torch.randn(1 << 16, device=DEV).square().sum()                # the program's own work, and a wait for it
                torch.cuda.synchronize()
            assert all(float(t) == 6 for t in ts)
            ends.append([norms] + [_flat(t) for t in (*ps, *(x for s in st for x in s if x is not None))])
        assert ends[0][0] == ends[1][0]
        for a, b in zip(ends[0][1:], ends[1][1:]):
            assert np.array_equal(a, b)


def test_a_step_on_another_stream_and_two_at_once():
    from igcn_cf_amd import ops
    rng = np.random.default_rng(10)
    sets = []
    for _ in range(4):
        p, g = _params((200003,), rng), _grads((200003,), rng)
        sets.append((p, g, _zeros8(p), torch.zeros((), device=DEV)))
    want = []
    for p, g, (m, v, s), t in sets:
        q, st, tt = p.clone(), _zeros8(p), t.clone()
        for _ in range(3):
            ops.adamw_step([q], [g], [st[0]], [st[1]], [tt], scales=[st[2]], max_grad_norm=1.0, **HYPER)
        want.append((q, *st))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for stream, (p, g, (m, v, s), t) in zip(streams, sets):
            with torch.cuda.stream(stream):
                ops.adamw_step([p], [g], [m], [v], [t], scales=[s], max_grad_norm=1.0, **HYPER)
    torch.cuda.synchronize()
    for (p, g, (m, v, s), t), w in zip(sets, want):
        assert torch.equal(p, w[0]) and torch.equal(m.view(torch.uint8), w[1].view(torch.uint8)) and torch.equal(v.view(torch.uint8), w[2].view(torch.uint8)) and torch.equal(s, w[3])


# ---- the optimizer -----------------------------------------------------------------------------------------------------------------
def _model(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(40, 64), torch.nn.Tanh(), torch.nn.Linear(64, 30)).to(DEV)


def _loss(model, k):
    x = torch.randn(50, 40, generator=torch.Generator().manual_seed(k)).to(DEV)
    return model(x).square().mean()


def test_optimizer_follows_the_formula_and_takes_another_adamws_state():
    """Against the step in 64 bits, fed the same gradients; and a run continued from a state_dict — torch's own AdamW's among them —
    goes on as the one it was taken from (float32 moments to one rounding a step of each: 1e-6 over 5 steps)."""
    from igcn_cf_amd.optim import AdamW
    model, other = _model(), _model()
    ours = AdamW(model.parameters(), **HYPER, max_grad_norm=0.05)
    theirs = torch.optim.AdamW(other.parameters(), **HYPER)
    for k in range(5):
        for m, o in ((model, ours), (other, theirs)):
            o.zero_grad()
            _loss(m, k).backward()
        want = torch.nn.utils.clip_grad_norm_(other.parameters(), 0.05)
        ours.step()
        theirs.step()
        assert abs(float(ours.grad_norm) / float(want) - 1) < 1e-5
    for a, b in zip(model.parameters(), other.parameters()):
        assert float((a - b).detach().abs().max()) < 1e-5 * 5
    third = _model()
    third.load_state_dict(other.state_dict())
    cont = AdamW(third.parameters(), **HYPER)
    cont.load_state_dict(theirs.state_dict())
    for k in range(5, 10):
        for m, o in ((third, cont), (other, theirs)):
            o.zero_grad()
            _loss(m, k).backward()
            o.step()
    for a, b in zip(third.parameters(), other.parameters()):
        assert float((a - b).detach().abs().max()) < 1e-4
    assert all(float(cont.state[p]['step']) == 10 for p in third.parameters())


@pytest.mark.parametrize('bits', [8, 32])
def test_a_saved_optimizer_goes_on_bit_for_bit(bits, tmp_path):
    from igcn_cf_amd.optim import AdamW
    model = _model().to(torch.bfloat16)
    groups = [{'params': [model[0].weight, model[0].bias]}, {'params': [model[2].weight, model[2].bias], 'lr': 1e-2, 'weight_decay': 0.}]
    opt = AdamW(groups, **HYPER, state_bits=bits, max_grad_norm=0.1, seed=5)

    def go(m, o, ks):
        for k in ks:
            o.zero_grad()
            x = torch.randn(50, 40, generator=torch.Generator().manual_seed(k)).to(DEV).to(torch.bfloat16)
            m(x).float().square().mean().backward()
            o.step()
    go(model, opt, range(3))
    torch.save({'model': model.state_dict(), 'opt': opt.state_dict()}, tmp_path / 'c.pt')
    saved = torch.load(tmp_path / 'c.pt', map_location=DEV, weights_only=True)
    again = _model(3).to(torch.bfloat16)
    again.load_state_dict(saved['model'])
    opt2 = AdamW([{'params': [again[0].weight, again[0].bias]}, {'params': [again[2].weight, again[2].bias]}], **HYPER, state_bits=bits, max_grad_norm=0.1, seed=5)
    opt2.load_state_dict(saved['opt'])
    for p, q in zip((q for g in opt.param_groups for q in g['params']), (q for g in opt2.param_groups for q in g['params'])):
        for name, value in opt.state[p].items():
            assert opt2.state[q][name].dtype == value.dtype and np.array_equal(_flat(opt2.state[q][name]), _flat(value))
        assert bits == 32 or opt.state[p]['exp_avg'].dtype == torch.float8_e4m3fn
    go(model, opt, range(3, 6))
    go(again, opt2, range(3, 6))
    for a, b in zip(model.parameters(), again.parameters()):
        assert torch.equal(a, b)
    size = sum(t.numel() * t.element_size() for p in model.parameters() for n, t in opt.state[p].items() if n != 'step')
    assert bits == 32 or size <= sum(2 * p.numel() + 8 * (p.numel() // 128 + 1) for p in model.parameters())


def test_parameters_without_gradient_and_gradients_in_another_order():
    from igcn_cf_amd.optim import AdamW
    a, b, c = (torch.nn.Parameter(torch.ones(6, 5, device=DEV)) for _ in range(3))
    opt = AdamW([a, b, c], lr=0.1, weight_decay=0.)
    a.grad = torch.arange(30., device=DEV).view(5, 6).t() + 1                         # transposed in memory
    c.grad = torch.ones(6, 5, device=DEV)
    version = a._version
    opt.step()
    assert a._version > version and torch.equal(b, torch.ones_like(b)) and not opt.state[b]
    assert torch.allclose(a, torch.full_like(a, 0.9), atol=1e-6) and torch.equal(opt.state[a]['exp_avg'].argmax(), a.grad.contiguous().argmax())
    opt.step(closure=lambda: None)
    assert float(opt.state[a]['step']) == 2


# ---- the trainers ------------------------------------------------------------------------------------------------------------------
def _trainer(name, hip_graph, bits, **kw):
    from igcn_cf_amd.dataset import SyntheticDataset
    from igcn_cf_amd.model import get_model
    from igcn_cf_amd.trainer import get_trainer
    torch.manual_seed(1)
    ds = SyntheticDataset({'name': 'SyntheticDataset', 'n_users': 600, 'n_items': 400, 'n_inter': 12000, 'device': DEV, 'seed': 3})
    model = get_model({'name': name, 'embedding_size': 64, 'n_layers': 2, 'dropout': 0.1, 'feature_ratio': 1., 'device': DEV}, ds)
    cfg = {'name': 'IGCNTrainer' if name == 'IGCN' else 'BPRTrainer', 'optimizer': 'AdamW', 'lr': 5e-3, 'l2_reg': 1e-4, 'aux_reg': 0.01, 'device': DEV,
           'n_epochs': 1, 'batch_size': 1024, 'topks': [20], 'hip_graph': hip_graph, 'state_bits': bits, 'weight_decay': 1e-3, 'max_grad_norm': 0.05, **kw}
    return ds, model, get_trainer(cfg, ds, model)


@pytest.mark.parametrize('name', ['MF', 'LightGCN', 'IGCN'])
@pytest.mark.parametrize('bits', [8, 32])
def test_trainers_take_the_step_by_name_captured_or_not(name, bits):
    """config 'optimizer': 'AdamW': captured and eager steps count and move alike (batch gradients come from float atomics, whose order
    differs from run to run, so the losses agree to 1e-3 rather than to the bit)."""
    ends = []
    for hip_graph in (True, False):
        ds, model, trainer = _trainer(name, hip_graph, bits)
        assert type(trainer.opt).__module__ == 'igcn_cf_amd.optim' and trainer._graph_wanted() == hip_graph
        model.train()
        losses = [trainer.train_one_epoch() for _ in range(2)]
        assert all(np.isfinite(losses))
        assert (trainer._graph is not None) == hip_graph
        steps = {float(s['step']) for s in trainer.opt.state.values()}
        assert len(trainer.opt.state) == len(list(model.parameters())) and len(steps) == 1
        ends.append((losses, steps))
    assert ends[0][1] == ends[1][1] and min(ends[0][1]) > 2
    assert all(abs(a - b) < 1e-3 for a, b in zip(ends[0][0], ends[1][0]))


def test_train_in_8_bits_clip_quantize_and_answer():
    """The operators as they are used together: LightGCN trained with 8-bit moments and clipped gradients, its item rows made 8-bit,
    the dense score block answered from them — every score within the codes' bound of the float32 block's."""
    ds, model, trainer = _trainer('LightGCN', True, 8)
    model.train()
    for _ in range(2):
        trainer.train_one_epoch()
    assert 0 < float(trainer.opt.grad_norm) < 1e3
    model.eval()
    users = torch.tensor([0, 5, 599, 5, 17], device=DEV)
    items = model.quantized_items()
    with torch.no_grad():
        want = model.predict(users).double()
        rep = model.get_rep()
    u, i = rep[users].double(), rep[ds.n_users:].double()
    eu, ei = u.abs().amax(1, keepdim=True) / 254, i.abs().amax(1, keepdim=True) / 254          # half a code step
    bound = eu * i.abs().sum(1) + u.abs().sum(1, keepdim=True) * ei.t() + 64 * eu * ei.t()
    for dtype in (torch.float32, torch.bfloat16):
        got = model.predict_i8(users, items, dtype=dtype)
        half = torch.finfo(dtype).eps / 2
        assert got.dtype == dtype and got.shape == (5, ds.n_items)
        slack = (half + 8 * 2.0 ** -24) * (want.abs() + bound) + 64 * 2.0 ** -24 * u.abs().sum(1, keepdim=True) * i.abs().amax(1)
        assert bool(((got.double() - want).abs() <= bound * (1 + 1e-5) + slack).all())
    assert torch.equal(model.predict_i8(users), model.predict_i8(users, items))


def test_refusals_leave_everything_as_it_was():
    from igcn_cf_amd import _lib, ops
    def lists(eight=False, shape=(40, 8)):
        ps = [torch.ones(shape, device=DEV), torch.ones(300, device=DEV)]
        gs = [torch.ones_like(p) for p in ps]
        if eight:
            ms, vs = ([torch.zeros_like(p, dtype=torch.uint8).view(d) for p in ps] for d in ops.MOMENT_DTYPES)
        else:
            ms, vs = ([torch.zeros_like(p) for p in ps] for _ in range(2))
        steps = [torch.zeros((), device=DEV) for _ in ps]
        scales = [torch.zeros((p.numel() + 127) // 128, 2, device=DEV) for p in ps]
        return dict(params=ps, grads=gs, exp_avgs=ms, exp_avg_sqs=vs, steps=steps, scales=scales if eight else None, lr=0.1)

    def change(name, at, value):
        def f(kw):
            kw[name][at] = value(kw) if callable(value) else value
        return f

    def setting(**new):
        return lambda kw: kw.update(new)
    buffer = torch.ones(700, device=DEV)
    both = [change('params', 1, lambda kw: kw['params'][0]), change('steps', 1, lambda kw: kw['steps'][0]), change('exp_avgs', 1, lambda kw: kw['exp_avgs'][0]),
            change('exp_avgs', 1, lambda kw: kw['exp_avg_sqs'][1].view(kw['exp_avgs'][1].dtype)), change('grads', 1, lambda kw: kw['params'][1]),
            lambda kw: kw.update(params=[buffer[:320].view(40, 8), buffer[319:619]]),
            change('grads', 0, torch.ones(8, 40, device=DEV)), change('grads', 0, torch.ones(8, 40, device=DEV).t()), change('grads', 0, torch.ones(40, 8, device=DEV, dtype=torch.float16)),
            change('grads', 0, torch.ones(40, 8)), change('grads', 0, torch.ones(40, 1, device=DEV).expand(40, 8)), change('grads', 0, None),
            change('params', 0, torch.ones(40, 8, device=DEV, dtype=torch.float64)), change('params', 0, torch.ones(40, 16, device=DEV)[:, ::2]),
            change('exp_avgs', 0, torch.zeros(320, device=DEV)), change('exp_avg_sqs', 1, torch.zeros(300, device=DEV, dtype=torch.bfloat16)),
            change('steps', 0, torch.zeros(2, device=DEV)), change('steps', 0, torch.zeros((), device=DEV, dtype=torch.int64)), change('steps', 0, torch.zeros(())),
            lambda kw: kw['steps'].pop(), setting(lr=-1.), setting(lr=torch.ones(2, device=DEV)), setting(lr=torch.ones(())), setting(lr=torch.ones((), device=DEV, dtype=torch.float64)),
            setting(betas=(0.9, 1.)), setting(eps=-1.), setting(weight_decay=float('nan')), setting(max_grad_norm=-1.), setting(max_grad_norm=float('nan')),
            setting(max_grad_norm=1., grad_norm=torch.ones(())), setting(max_grad_norm=1., grad_norm=2.)]
    eight_only = [change('scales', 0, torch.zeros(2, 2, device=DEV)), change('scales', 1, torch.zeros(3, 2, device=DEV, dtype=torch.float64)), change('scales', 0, torch.zeros(2, 3, device=DEV).t()),
                  lambda kw: kw['scales'].pop(), setting(scales=None), change('exp_avgs', 0, torch.zeros(40, 8, device=DEV)), change('scales', 1, lambda kw: kw['scales'][0])]
    for eight in (False, True):
        for i, spoil in enumerate(both + (eight_only if eight else [])):
            kw = lists(eight)
            spoil(kw)
            with pytest.raises(_lib.IgcnError):
                ops.adamw_step(**kw)
                print('not refused:', eight, i)
            for name, want in (('params', 1.), ('steps', 0.)):
                for t in kw[name]:
                    assert bool((t.double() == want).all()), (eight, i, name)
        kw = lists(eight)
        kw['lr'], kw['betas'] = np.float32(0.1), (np.float32(0.9), np.float64(0.999))                       # numbers of any make
        ops.adamw_step(seed=np.int64(-3), max_grad_norm=np.float32(1.), **kw)
        shared = lists(eight, shape=(300,))
        shared['grads'][1] = shared['grads'][0]                                                            # gradients may be one
        ops.adamw_step(**shared)
        assert bool((shared['params'][0] < 1).all()) and torch.equal(shared['params'][0], shared['params'][1])
    for gs in ([torch.ones(3)], [torch.ones(3, device=DEV).double()], [torch.ones(1, device=DEV).expand(3)], [None], [torch.ones(4, 4, device=DEV)[:, 1]]):
        with pytest.raises(_lib.IgcnError):
            ops.grad_norm(gs)


@pytest.mark.parametrize('eight', [False, True])
def test_elements_past_32_bits(eight):
    """More than 2^31 elements (2^32 with 8-bit moments): the last ones are stepped like a tensor of their own, the ones before are not touched twice."""
    from igcn_cf_amd import ops
    n, tail = (2 ** 32 if eight else 2 ** 31) + 1000, 1000
    p, g = torch.ones(n, dtype=torch.bfloat16, device=DEV), torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g[-tail:] = torch.randn(tail, device=DEV, generator=torch.Generator(DEV).manual_seed(3)).to(torch.bfloat16)
    g[:tail] = g[-tail:]
    if eight:
        m, v, scales = _zeros8(p)
    else:
        m, v, scales = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), None
    step = torch.zeros((), device=DEV)
    norm = ops.adamw_step([p], [g], [m], [v], [step], lr=0.25, weight_decay=0., eps=0.5, max_grad_norm=1e6, scales=[scales] if eight else None)
    assert abs(float(norm) - float(g[-tail:].double().norm()) * 2 ** 0.5) <= 1e-6 * float(norm)
    x = g[-tail:].double()
    want = 1 - 0.25 * x / (x.abs() + 0.5)                                            # the first step: m / c1 = g, v / c2 = g^2 (its float32 roundings: well under 1e-5)
    for part in (slice(0, tail), slice(n - tail, n)):
        assert bool(((p[part].double() - want).abs() <= HALF_STEP[torch.bfloat16] * want.abs() + 1e-5).all())
    assert bool((p[tail:2 * tail] == 1).all()) and bool((p[-2 * tail:-tail] == 1).all())
    if eight:
        block = torch.arange(n - tail, n, device=DEV) // 128                         # code steps: an eighth of the value, 2^-9 of the scale at least
        s = scales[block, 0].double()
        assert bool(((m[-tail:].float().double() * s - 0.1 * x).abs() <= 0.13 * (0.1 * x).abs() + s * 2.0 ** -9 * 1.01).all())
    else:
        assert bool(((m[-tail:].double() - 0.1 * x).abs() <= 1e-6 * x.abs()).all())


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('betas', [(0., 0.999), (0.9, 0.), (0., 0.), (0.1, 0.2), (0.49, 0.51), (0.5, 0.5), (0.51, 0.49), (0.999, 0.3), (1e-6, 1e-6)])
def test_every_beta_leaves_what_its_moment_keeps(betas, eight):
    """Old averages far above or far below the new gradient, for betas over the whole range: an average keeps beta of itself and takes
    1 - beta of the new value, each to a few roundings of its own size.  u = 2^-24 a rounding: beta, 1 - beta, two products and the sum round,
    so m is within 4 u (b |m| + a |x|) and v within 5 u (b v + a x^2); the update adds sqrt, reciprocal (1 ulp = 2 u each), its
    factors and products: 16 u of its size in all.  8-bit codes hold a moment to an eighth / a quarter, or a step of their block."""
    from igcn_cf_amd import ops
    u, n = 2.0 ** -24, 700
    hyper = dict(HYPER, betas=betas)
    for old_m, old_v, size in ((0., 1., 1e-4), (1., 1., 1e-4), (1., 1e-8, 1e3), (1e-3, 1e-12, 1e-3), (0., 0., 1.)):
        rng = np.random.default_rng(3)
        g = torch.from_numpy((size * rng.standard_normal(n)).astype(np.float32)).to(DEV)
        p, t = _params((n,), rng), torch.full((), 4., device=DEV)
        m, v = torch.full((n,), old_m, device=DEV), torch.full((n,), old_v, device=DEV)
        if eight:
            s = torch.tensor([[old_m / 448 or 1., old_v / 57344 or 1.]], device=DEV).repeat(-(-n // 128), 1)
            m8 = torch.full((n,), 126 if old_m else 0, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
            v8 = torch.full((n,), 123 if old_v else 0, dtype=torch.uint8, device=DEV).view(torch.float8_e5m2)
            m, v = m8.float() * s[:, 0].repeat_interleave(128)[:n], v8.float() * s[:, 1].repeat_interleave(128)[:n]
        p0, m0, v0, x = _flat(p), _flat(m), _flat(v), _flat(g)
        ops.adamw_step([p], [g], [m8 if eight else m], [v8 if eight else v], [t], scales=[s] if eight else None, **hyper)
        (b1, b2), c1, c2 = betas, 1 - betas[0] ** 5, 1 - betas[1] ** 5
        size_m, size_v = b1 * np.abs(m0) + (1 - b1) * np.abs(x), b2 * v0 + (1 - b2) * x * x
        m1, v1 = b1 * m0 + (1 - b1) * x, size_v
        if eight:
            sm, sv = (s[:, j].double().repeat_interleave(128)[:n].cpu().numpy() for j in (0, 1))
            assert (np.abs(_flat(m8.float()) * sm - m1) <= np.abs(m1) / 8 + sm * 2.0 ** -9 + 8 * u * size_m).all(), (old_m, size)
            assert (np.abs(_flat(v8.float()) * sv - v1) <= v1 / 4 + sv * 2.0 ** -16 + 8 * u * size_v).all(), (old_v, size)
        else:
            assert (np.abs(_flat(m) - m1) <= 4 * u * size_m).all(), (old_m, size)
            assert (np.abs(_flat(v) - v1) <= 5 * u * size_v).all(), (old_v, size)
        denom = np.sqrt(v1 / c2) + hyper['eps']
        step = hyper['lr'] / c1
        want = p0 * (1 - hyper['lr'] * hyper['weight_decay']) - step * m1 / denom
        assert (np.abs(_flat(p) - want) <= 4 * u * np.abs(p0) + 16 * u * step * size_m / denom).all(), (old_m, old_v, size)


@pytest.mark.parametrize('eight', [False, True])
def test_gradients_whose_squares_alone_pass_float32(eight):
    """(1 - beta2) x^2 is a float32 number up to |x| = 5.8e20 at beta2 = 0.999, x^2 up to 1.8e19 only: what is held is the formula's."""
    from igcn_cf_amd import ops
    g = torch.tensor([1e19, -3e19, 1e20, -5e20], device=DEV)
    for old in (0., 1e30):
        p, t = torch.zeros(4, device=DEV), torch.zeros((), device=DEV)
        m, v, s = torch.zeros(4, device=DEV), torch.full((4,), old, device=DEV), None
        if eight:
            m, v, s = _zeros8(p)
        ops.adamw_step([p], [g], [m], [v], [t], scales=[s] if eight else None, **HYPER)
        x = _flat(g)
        v1 = 0.999 * (0. if eight else old) + 0.001 * x * x
        if eight:
            assert (np.abs(_flat(v.float()) * float(s[0, 1]) - v1) <= v1 / 4 + float(s[0, 1]) * 2.0 ** -16).all()
        else:
            assert (np.abs(_flat(v) - v1) <= 5 * 2.0 ** -24 * v1).all()
        want = -HYPER['lr'] * x / np.sqrt(v1 / 0.001)
        assert (np.abs(_flat(p) - want) <= 24 * 2.0 ** -24 * np.abs(want)).all()
    if not eight:                                                                    # an infinite average stays one and moves nothing
        p, m, v = torch.ones(4, device=DEV), torch.ones(4, device=DEV), torch.full((4,), float('inf'), device=DEV)
        ops.adamw_step([p], [torch.ones(4, device=DEV)], [m], [v], [torch.zeros((), device=DEV)], lr=1e-3, weight_decay=0.)
        assert bool(torch.isinf(v).all()) and bool((p == 1).all())


def test_a_small_eps_and_second_moments_below_float32s_normal_numbers():
    """eps is any number from 0 on, and v may be as small as float32 has them (2^-149): the update is step m / (sqrt(v / c2) + eps) of the
    moments the step left, its roundings as ever (sqrt and reciprocal 1 ulp = 2 u each, four products, a constant each: 12 u), where neither
    is lost below 2^-126 (4.6e-10 is where the kernels change over).  p starts at zero and nothing decays: what is there is the update."""
    from igcn_cf_amd import ops
    u = 2.0 ** -24
    old = torch.tensor([2.0 ** e for e in (-149, -148, -145, -140, -133, -127, -126, -125, -110, -101, -100, -99, -90, -40, 0)] + [0.], device=DEV)
    for eps in (0., 2.0 ** -149, 1e-42, 1e-40, 2.0 ** -127, 1.2e-38, 1e-35, 1e-30, 1e-20, 4.5e-10, 4.7e-10, 1e-8):
        for near in (1., 2.0 ** -20):
            p, g, t = torch.zeros(16, device=DEV), torch.zeros(16, device=DEV), torch.full((), 9., device=DEV)
            m = (old.double().sqrt().clamp(min=max(float(np.float32(eps)), 2.0 ** -120)) * near).float()       # updates of ordinary size
            v = old.clone()
            ops.adamw_step([p], [g], [m], [v], [t], lr=1e-3, betas=(0.9, 0.999), eps=eps, weight_decay=0.)
            m1, v1, eps32 = _flat(m), _flat(v), float(np.float32(eps))
            with np.errstate(divide='ignore', invalid='ignore'):
                want = -1e-3 / (1 - 0.9 ** 10) * m1 / (np.sqrt(v1 / (1 - 0.999 ** 10)) + eps32)
            got = _flat(p)
            wide = np.abs(want) > np.finfo(np.float32).max
            assert (np.isinf(got) == (wide | np.isinf(want))).all(), (eps, near, got)
            fine = np.isfinite(want) & ~wide
            assert (np.abs(got[fine] - want[fine]) <= 12 * u * np.abs(want[fine]) + 2.0 ** -149).all(), (eps, near, got, want)
    p, z = torch.zeros(3, device=DEV), [torch.zeros(3, device=DEV) for _ in range(3)]
    ops.adamw_step([p], [z[0]], [z[1]], [z[2]], [torch.zeros((), device=DEV)], lr=1e-3, eps=1e-40)
    assert not p.any()                                                              # 0 / eps


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('n', [64, 20003])
@pytest.mark.parametrize('eps', [0., 1e-42, 1e-30, 1e-8])
def test_first_steps_from_gradients_whose_squares_are_hardly_there(n, eight, eps):
    """A first step moves a parameter by lr g / (|g| + eps), whatever the size of g, in one launch and in two.  v = 0.001 g^2 may lie below 2^-126,
    where float32 has steps of 2^-149: two such roundings of v, halved by the root, beside 16 u of the update (u = 2^-24)."""
    from igcn_cf_amd import ops
    u = 2.0 ** -24
    g = torch.pow(2.0, -40 - 24 * torch.rand(n, device=DEV, generator=torch.Generator(DEV).manual_seed(n)))
    g[::3] *= -1
    for dtype in (torch.float32, torch.bfloat16):
        p, gd, t = torch.zeros(n, device=DEV, dtype=dtype), g.to(dtype), torch.zeros((), device=DEV)
        m, v, s = _zeros8(p) if eight else (torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), None)
        ops.adamw_step([p], [gd], [m], [v], [t], scales=[s] if eight else None, lr=1e-3, betas=(0.9, 0.999), eps=eps)
        x = _flat(gd)
        want = -1e-3 * x / (np.abs(x) + float(np.float32(eps)))
        off = (16 * u + 2.0 ** -149 / (0.001 * x * x)) * np.abs(want)
        assert (np.abs(_flat(p) - want) <= off + HALF_STEP[dtype] * (np.abs(want) + off)).all(), (dtype, n, eps)


@pytest.mark.parametrize('name', ['MF', 'LightGCN', 'IGCN'])
def test_a_model_cut_by_columns_is_clipped_by_the_norm_of_all_its_columns(name):
    """Two column slices trained side by side (a thread each, the all-reduce a sum over both) hold the moments of the unsharded trainer:
    clipping scales every column by the one factor.  The slices' own norms are far apart, so a factor of a slice's own would be off by
    1.2 and more in one of them; gradients agree to the order of their float32 sums (1e-4 of the largest is far above it)."""
    import threading
    from igcn_cf_amd.dataset import SyntheticDataset
    from igcn_cf_amd.dist import column_shard_model
    from igcn_cf_amd.model import get_model
    from igcn_cf_amd.trainer import get_trainer
    ds = SyntheticDataset({'name': 'SyntheticDataset', 'n_users': 300, 'n_items': 200, 'n_inter': 5000, 'device': DEV, 'seed': 3})
    mcfg = {'name': name, 'embedding_size': 32, 'n_layers': 2, 'dropout': 0., 'feature_ratio': 1., 'device': DEV}
    tcfg = {'name': 'IGCNTrainer' if name == 'IGCN' else 'BPRTrainer', 'optimizer': 'AdamW', 'lr': 1e-3, 'l2_reg': 1e-2, 'aux_reg': 0.1, 'device': DEV,
            'n_epochs': 1, 'batch_size': 256, 'topks': [20], 'weight_decay': 0., 'max_grad_norm': 1e-3, 'hip_graph': False}
    torch.manual_seed(4)
    whole = get_model(mcfg, ds)
    with torch.no_grad():
        for k, p in whole.state_dict().items():
            if p.dim() == 2:
                p[:, :16] *= 5.
    state = {k: v.detach().clone() for k, v in whole.state_dict().items()}
    batches = [torch.stack([torch.randint(0, hi, (256,), generator=torch.Generator().manual_seed(i)) for hi in (300, 200, 200)], 1).to(DEV) for i in range(3)]

    def go(trainer):
        trainer.model.train()
        for b in batches:
            if name == 'IGCN':
                trainer.igcn_step(b, b)
            else:
                trainer.bpr_step(b)
        torch.cuda.synchronize()
    plain = get_trainer(tcfg, ds, whole)
    go(plain)
    assert float(plain.opt.grad_norm) > 3e-3                                         # (clipping does something)
    barrier, slots, errors = threading.Barrier(2, timeout=60), [None, None], []

    def reduce_of(rank):
        def reduce(t):
            slots[rank] = t.clone()
            barrier.wait()
            total = slots[0] + slots[1]
            barrier.wait()
            return t.copy_(total)
        return reduce
    trainers = [get_trainer(tcfg, ds, column_shard_model(mcfg, ds, r, 2, full_state=state, reduce_fn=reduce_of(r))) for r in range(2)]

    def rank(r):
        try:
            go(trainers[r])
        except Exception as e:                                                       # noqa: BLE001 (shown below)
            errors.append(e)
            barrier.abort()
    threads = [threading.Thread(target=rank, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for k, p in dict(whole.named_parameters()).items():
        for what in ('exp_avg', 'exp_avg_sq'):
            want = plain.opt.state[p][what]
            got = torch.cat([tr.opt.state[dict(tr.model.named_parameters())[k]][what] for tr in trainers], -1)
            assert float((got - want).abs().max()) <= 1e-4 * float(want.abs().max()), (k, what)
    for tr in trainers:
        assert abs(float(tr.opt.grad_norm) / float(plain.opt.grad_norm) - 1) < 1e-4


@pytest.mark.parametrize('name', ['MF', 'LightGCN'])
def test_the_norm_is_the_last_steps_replayed_or_eager(name):
    """Full batches replay a captured step, a shorter one runs eagerly: grad_norm is that of whichever ran last, in one tensor throughout.
    Nothing moves (lr 0), so a batch's norm is the same whenever it runs, to the order of its float32 sums."""
    ds, model, trainer = _trainer(name, True, 32)
    for group in trainer.opt.param_groups:
        group['lr'] = 0.
    model.train()
    if name == 'MF':
        step, batches = trainer.flat_step, lambda n: next(iter(trainer.sampler.epoch_node_batches(n, 0)))
    else:
        step, batches = trainer.node_step, lambda n: next(iter(trainer.sampler.epoch_node_batches(n, ds.n_users)))
    full, short = batches(1024).clone(), batches(40).clone()
    step(full)
    held, at_full = trainer.opt.grad_norm, float(trainer.opt.grad_norm)
    step(short)
    at_short = float(trainer.opt.grad_norm)
    assert abs(at_short / at_full - 1) > 0.01
    for _ in range(2):
        step(full)
        assert abs(float(trainer.opt.grad_norm) / at_full - 1) < 1e-4
        step(short)
        assert abs(float(trainer.opt.grad_norm) / at_short - 1) < 1e-4
    assert trainer._graph is not None and trainer.opt.grad_norm is held


def test_a_norm_goes_where_it_is_asked_to():
    from igcn_cf_amd import _lib, ops
    rng = np.random.default_rng(12)
    gs = [_grads(s, rng) for s in ((3, 50), (70001,))]
    want, out = ops.grad_norm(gs), torch.zeros(1, device=DEV)
    assert ops.grad_norm(gs, out=out) is out and out[0] == want
    assert ops.grad_norm([], out=out) is out and float(out) == 0.
    for n in (1, 2):                                                                 # one launch, and more
        for given in (None, torch.full((), 7., device=DEV)):
            p = [torch.ones_like(g) for g in gs[:n]]
            m, v, t = [torch.zeros_like(g) for g in p], [torch.zeros_like(g) for g in p], [torch.zeros((), device=DEV) for _ in p]
            out.fill_(-1.)
            got = ops.adamw_step(p, gs[:n], m, v, t, lr=0.1, max_grad_norm=1., grad_norm=given, norm_out=out)
            assert (got is out and out[0] == ops.grad_norm(gs[:n])) if given is None else (got is given and float(out) == -1.)
    for bad in (torch.zeros(()), torch.zeros(2, device=DEV), torch.zeros((), dtype=torch.float64, device=DEV), 1., t[0]):
        with pytest.raises(_lib.IgcnError):
            ops.adamw_step(p, gs, m, v, t, lr=0.1, max_grad_norm=1., norm_out=bad)
        if bad is not t[0]:
            with pytest.raises(_lib.IgcnError):
                ops.grad_norm(gs, out=bad)
    with pytest.raises(_lib.IgcnError):
        ops.adamw_step(p, gs, m, v, t, lr=p[0][0, :1], max_grad_norm=1.)
    with pytest.raises(_lib.IgcnError):
        ops.adamw_step(p, gs, m, v, t, lr=0.1, max_grad_norm=1., grad_norm=t[1])


def test_a_step_without_gradients_has_norm_zero():
    from igcn_cf_amd.optim import AdamW
    w = torch.nn.Parameter(torch.ones(3, device=DEV))
    opt = AdamW([w], max_grad_norm=1.)
    w.grad = torch.full((3,), 2., device=DEV)
    opt.step()
    assert abs(float(opt.grad_norm) - 12 ** 0.5) < 1e-6
    w.grad = None
    opt.step()
    assert float(opt.grad_norm) == 0.


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_a_run_of_torchs_adamw_in_16_bits_goes_on(dtype):
    """Its moments are in the parameter's type, one parameter is transposed in memory and one saved moment is not: the next step is the
    formula's from the saved values (where torch's own steps left the parameter finite: 1e-8 is 0 in float16, and some of its second moments are)."""
    from igcn_cf_amd.optim import AdamW
    rng = np.random.default_rng(14)
    ps = [torch.nn.Parameter(_params((33, 20), rng, dtype)), torch.nn.Parameter(_params((20, 33), rng, dtype).t())]
    theirs = torch.optim.AdamW(ps, **HYPER)
    for _ in range(3):
        for p in ps:
            p.grad = _grads((33, 20), rng, dtype)
        theirs.step()
    saved = theirs.state_dict()
    saved['state'][1]['exp_avg'] = saved['state'][1]['exp_avg'].contiguous()
    ours = AdamW(ps, **HYPER)
    ours.load_state_dict(saved)
    before = [(p.detach().clone(), ours.state[p]['exp_avg'].clone(), ours.state[p]['exp_avg_sq'].clone()) for p in ps]
    for (p0, m0, v0), i in zip(before, range(2)):
        assert m0.dtype == torch.float32 and torch.equal(m0, saved['state'][i]['exp_avg'].float()) and torch.equal(v0, saved['state'][i]['exp_avg_sq'].float())
    gs = [torch.empty_like(p).copy_(_grads((33, 20), rng, dtype)) for p in ps]
    for p, g in zip(ps, gs):
        p.grad = g
    ours.step()
    for p, g, (p0, m0, v0) in zip(ps, gs, before):
        fine = torch.isfinite(p0)
        assert bool(torch.isclose(p[~fine], p0[~fine], equal_nan=True).all()) and bool(fine.any())
        _check32(p0[fine], g[fine], m0[fine], v0[fine], 4, p[fine], ours.state[p]['exp_avg'][fine], ours.state[p]['exp_avg_sq'][fine])


@pytest.mark.parametrize('name,bits', [('MF', 32), ('LightGCN', 8), ('LightGCN', 32)])
def test_captured_steps_follow_a_state_that_is_loaded_between_them(name, bits):
    """Back to a checkpoint in mid-run: steps, a save, more steps, model and optimizer loaded, more steps — captured like eager.  Moments are what the
    restored ones lead to (their steps go on from the checkpoint's); gradients come from float atomics, so they agree to their sums' order."""
    import copy
    ends = []
    for hip_graph in (True, False):
        ds, model, trainer = _trainer(name, hip_graph, bits)
        if name == 'MF':
            step, draw = trainer.flat_step, lambda n: trainer.sampler.epoch_node_batches(n, 0)
        else:
            step, draw = trainer.node_step, lambda n: trainer.sampler.epoch_node_batches(n, ds.n_users)
        batches, short = [b.clone() for _, b in zip(range(6), draw(1024))], next(draw(40)).clone()
        for b in batches + [short]:
            users, items = b.view(3, -1)[0], b.view(3, -1)[1:] - (0 if name == 'MF' else ds.n_users)
            assert 0 <= int(users.min()) and int(users.max()) < ds.n_users and 0 <= int(items.min()) and int(items.max()) < ds.n_items
        model.train()
        for b in batches[:3]:
            step(b)
        saved = copy.deepcopy((model.state_dict(), trainer.opt.state_dict()))
        first = trainer._graph
        for b in batches[3:]:
            step(b)
        assert trainer._graph is first and (first is not None) == hip_graph
        held = [dict(s) for s in trainer.opt.state.values()]                          # (the old memory stays: nothing may still go there)
        before = [{k: v.clone() for k, v in s.items()} for s in held]
        model.load_state_dict(saved[0])
        trainer.opt.load_state_dict(saved[1])
        for b in batches[3:] * 2:
            step(b)
            step(short)                                                              # eager
        torch.cuda.synchronize()
        for h, b in zip(held, before):
            assert all(torch.equal(h[k].view(torch.uint8) if h[k].dim() else h[k], b[k].view(torch.uint8) if b[k].dim() else b[k]) for k in h)
        assert {float(s['step']) for s in trainer.opt.state.values()} == {15.}
        ends.append([trainer.opt.state[p]['exp_avg'].float() if bits == 32 else
                     trainer.opt.state[p]['exp_avg'].float().reshape(-1) * trainer.opt.state[p]['scales'][:, 0].repeat_interleave(128)[:p.numel()]
                     for p in model.parameters()])
    for a, b in zip(*ends):
        assert float((a - b).abs().mean()) <= 1e-2 * float(b.abs().max())


def test_a_captured_step_reads_a_device_rate_anew():
    """A learning rate on the GPU is read by the replays: changing it neither captures again nor waits for the GPU, another tensor in its place does
    capture.  Rate 0 moves nothing (no decay at that rate either)."""
    ds, model, trainer = _trainer('MF', True, 32)
    lr = torch.full((), 1e-2, device=DEV)
    trainer.opt.param_groups[0]['lr'] = lr
    model.train()
    batch = next(iter(trainer.sampler.epoch_node_batches(1024, 0))).clone()
    trainer.flat_step(batch)
    first, key = trainer._graph, trainer._graph_key()
    lr.zero_()
    assert trainer._graph_key() == key and all(type(k) is not torch.Tensor for k in key)
    before = [p.detach().clone() for p in model.parameters()]
    trainer.flat_step(batch)
    assert trainer._graph is first and all(torch.equal(p, b) for p, b in zip(model.parameters(), before))
    lr.fill_(1e-2)
    trainer.flat_step(batch)
    assert trainer._graph is first and not any(torch.equal(p, b) for p, b in zip(model.parameters(), before))
    trainer.opt.param_groups[0]['lr'] = torch.full((), 1e-3, device=DEV)
    trainer.flat_step(batch)
    assert trainer._graph is not first
