"""What the optimizer step and the 8-bit operators refuse, without a GPU: the Python entry points on tensors they do not take, the C
entry points by error code before anything is launched, and the plain forms the GPU tests rest on."""
import array
import ctypes as C

import numpy as np
import pytest
import torch

from igcn_cf_amd import _lib, ops
from igcn_cf_amd.optim import AdamW
from tests import adamw_oracle as A


def test_python_entry_points_refuse_cpu_tensors_and_bad_settings():
    p = torch.zeros(4, 4)
    t = torch.zeros(())
    for call in (lambda: ops.adamw_step([p], [p], [p.clone()], [p.clone()], [t], lr=1e-3), lambda: ops.grad_norm([p]), lambda: ops.quantize_rows_i8(p),
                 lambda: ops.dequantize_rows_i8(p.to(torch.int8), t), lambda: ops.matmul_i8(p.to(torch.int8), t, p.to(torch.int8), t), lambda: ops.linear_i8(p, p, t),
                 lambda: ops.adamw_step([p], [], [], [], [], lr=1e-3), lambda: ops.adamw_step([], [], [], [], [], lr=1e-3, max_grad_norm=0.),
                 lambda: ops.adamw_step([], [], [], [], [], lr=-1.), lambda: ops.adamw_step([], [], [], [], [], lr=1e-3, betas=(0.9, 1.0))):
        with pytest.raises(_lib.IgcnError):
            call()
    assert ops.adamw_step([], [], [], [], [], lr=1e-3) is None
    w = torch.nn.Parameter(p)
    for kw in (dict(lr=-1.), dict(betas=(1., 0.9)), dict(eps=-1.), dict(weight_decay=-1.), dict(state_bits=16), dict(max_grad_norm=0.)):
        with pytest.raises(ValueError):
            AdamW([w], **kw)
    w.grad = torch.zeros(4, 4)
    with pytest.raises(_lib.IgcnError):
        AdamW([w]).step()


def _table(count=1, **kw):
    """igcn_adamw_tensor rows as int64 words; pointers that are aligned and never followed."""
    f = dict(param=0x1000, grad=0x2000, m=0x3000, v=0x4000, scales=0x5000, step=0x6000, n=256, dtype=0, grad_dtype=0)
    f.update(kw)
    row = [f['param'], f['grad'], f['m'], f['v'], f['scales'], f['step'], f['n'], f['dtype'] | f['grad_dtype'] << 32]
    return array.array('q', row * count)


def test_the_c_step_and_norm_reject_bad_arguments_before_any_launch():
    L = _lib.lib()

    def step(t, n=1, bits=32, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.01, mx=0., ni=None, no=None, ws=0x100):
        return L.igcn_adamw_step(t.buffer_info()[0] if t is not None else None, n, bits, lr, None, b1, b2, eps, wd, mx, ni, no, 0, ws, None)
    assert step(None) == -1 and step(_table(), n=-1) == -2
    assert step(_table(), bits=16) == -4
    for kw in (dict(lr=-1.), dict(lr=float('nan')), dict(b1=1.), dict(b2=-0.1), dict(eps=-1.), dict(wd=-1.), dict(mx=-1.), dict(mx=float('nan'))):
        assert step(_table(), **kw) == -4, kw
    assert step(_table(), ws=None) == -1 and step(_table(), ws=0x104) == -3 and step(_table(), mx=1.) == -1 and step(_table(), mx=1., no=0x102) == -3
    for kw in (dict(param=0), dict(grad=0), dict(m=0), dict(v=0), dict(step=0)):
        assert step(_table(**kw)) == -1, kw
    assert step(_table(scales=0), bits=8) == -1
    assert step(_table(dtype=3)) == -4 and step(_table(dtype=0, grad_dtype=1)) == -4 and step(_table(dtype=1, grad_dtype=2)) == -4
    for kw in (dict(param=0x1002), dict(grad=0x2001), dict(m=0x3002), dict(step=0x6002), dict(scales=0x5002), dict(dtype=1, param=0x1001, grad_dtype=1)):
        assert step(_table(**kw)) == -3, kw
    bad = _table()
    bad[6] = -5
    assert step(bad) == -2
    assert L.igcn_adamw_workspace_bytes(bad.buffer_info()[0], 1) == -1
    assert step(None, n=0) == 0                                                       # nothing to do
    one, other, lots = _table(), _table(grad_dtype=7), _table(200)                    # (held: the calls get their addresses)
    assert L.igcn_grad_norm(None, 0, None, 0x100, None) == -1 and L.igcn_grad_norm(one.buffer_info()[0], 1, 0x102, 0x100, None) == -3
    assert L.igcn_grad_norm(other.buffer_info()[0], 1, 0x100, 0x100, None) == -4
    few, many = L.igcn_adamw_workspace_bytes(one.buffer_info()[0], 1), L.igcn_adamw_workspace_bytes(lots.buffer_info()[0], 200)
    assert 0 < few < many


def test_the_struct_of_a_tensor_is_laid_out_as_the_binding_fills_it(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = ['param', 'grad', 'exp_avg', 'exp_avg_sq', 'scales', 'step', 'n', 'dtype', 'grad_dtype']
    src = tmp_path / 'layout.c'
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "igcn_hip.h"\nint main(void) {\n'
                   + ''.join('    printf("%%zu ", offsetof(igcn_adamw_tensor, %s));\n' % f for f in names)
                   + '    printf("%zu %d %d\\n", sizeof(igcn_adamw_tensor), IGCN_ADAMW_BLOCK, IGCN_MAX_I8_DEPTH);\n    return 0;\n}\n')
    subprocess.run(['gcc', '-std=c99', '-Wall', '-Werror', '-I', os.path.join(root, 'include'), str(src), '-o', str(tmp_path / 'layout')], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / 'layout')], check=True, stdout=subprocess.PIPE).stdout.split()]
    assert got == [0, 8, 16, 24, 32, 40, 48, 56, 60, 64, ops.ADAMW_BLOCK, ops.MAX_I8_DEPTH]


def test_the_c_8_bit_entry_points_reject_bad_arguments_before_any_launch():
    L = _lib.lib()
    P = 0x1000

    def quantize(x=P, dtype=0, ldx=64, rows=4, k=64, q=P, ldq=64, s=P):
        return L.igcn_quantize_rows_i8(x, dtype, ldx, rows, k, q, ldq, s, None)

    def back(q=P, ldq=64, s=P, rows=4, k=64, y=P, dtype=0, ldy=64):
        return L.igcn_dequantize_rows_i8(q, ldq, s, rows, k, y, dtype, ldy, None)

    def product(a=P, lda=64, sa=P, b=P, ldb=64, sb=P, bias=None, m=4, n=8, k=64, y=P, dtype=0, ldy=8):
        return L.igcn_matmul_i8(a, lda, sa, b, ldb, sb, bias, m, n, k, y, dtype, ldy, None)
    assert quantize(dtype=5) == -4 and quantize(rows=-1) == -2 and quantize(ldx=63) == -2 and quantize(ldq=1) == -2 and quantize(k=-1) == -2
    assert quantize(x=None) == -1 and quantize(q=None) == -1 and quantize(s=None) == -1 and quantize(x=0x1002) == -3 and quantize(x=0x1001, dtype=1) == -3 and quantize(s=0x1001) == -3
    assert quantize(rows=0, x=None) == 0
    assert back(dtype=-1) == -4 and back(ldy=3) == -2 and back(q=None) == -1 and back(s=None) == -1 and back(y=None) == -1 and back(y=0x1002) == -3 and back(k=0, q=None) == 0
    assert product(dtype=3) == -4 and product(m=-1) == -2 and product(lda=1) == -2 and product(ldb=1) == -2 and product(ldy=7) == -2
    assert product(k=131072, lda=1 << 20, ldb=1 << 20) == -4
    for kw in (dict(a=None), dict(b=None), dict(sa=None), dict(sb=None), dict(y=None)):
        assert product(**kw) == -1, kw
    assert product(y=0x1002) == -3 and product(sa=0x1002) == -3 and product(bias=0x1001) == -3 and product(m=0, a=None) == 0 and product(n=0, ldy=0) == 0


def test_the_plain_codes_are_those_torch_reads_and_round_both_ways():
    """decode() against torch's own float8 types over all finite codes; encode() with u just under 1 and just over 0 gives the neighbours."""
    codes = np.arange(256, dtype=np.uint8)
    for dtype, mantissa, bias in ((torch.float8_e4m3fn, 3, 7), (torch.float8_e5m2, 2, 15)):
        want = torch.from_numpy(codes).view(dtype).float().numpy()
        fine = np.isfinite(want)
        assert np.array_equal(A.decode(codes, mantissa, bias)[fine], want[fine]) and fine.sum() >= 248
    x = np.abs(np.random.default_rng(0).standard_normal(1280)).astype(np.float32)
    x[::128] = 10.
    low, s, _ = A.encode(x, np.zeros(1280, np.int64), 3, 7, 448.)
    high, _, _ = A.encode(x, np.full(1280, 65535), 3, 7, 448.)
    scale = np.repeat(s, 128).astype(np.float64)
    down, up = (A.decode(c.astype(np.uint8), 3, 7) * scale for c in (low, high))
    assert (down <= x * (1 + 1e-6)).all() and (up >= x * (1 - 1e-6)).all() and ((high - low) <= 1).all() and (high[::128] == 126).all()
    assert len({int(h) for h in A.hashes(1000, 7, 0, 1)}) > 990 and not np.array_equal(A.hashes(8, 7, 0, 1), A.hashes(8, 7, 1, 1))


def test_dense_orders_are_told_from_views_with_gaps():
    x = torch.zeros(6, 8, 10)
    for t in (x, x.transpose(0, 2), x[2], x[:, :1].squeeze(1)[1], x.reshape(-1)[3:7], torch.zeros(()), torch.zeros(0, 3)):
        assert ops._dense(t)
    for t in (x[:, 1], x[..., :3], x[::2], torch.zeros(1).expand(5)):
        assert not ops._dense(t)
    assert ops._same_order(x.transpose(0, 1), torch.empty_like(x.transpose(0, 1))) and not ops._same_order(x.transpose(0, 2), torch.zeros(10, 8, 6))


def test_the_c_step_refuses_shared_memory_and_tensors_too_long():
    L = _lib.lib()

    def step(*tables, bits=32):
        t = array.array('q')
        for x in tables:
            t.extend(x)
        return L.igcn_adamw_step(t.buffer_info()[0], len(tables), bits, 1e-3, None, 0.9, 0.999, 1e-8, 0.01, 0., None, None, 0, 0x100, None)
    far = dict(param=0x11000, m=0x13000, v=0x14000, scales=0x15000, step=0x16000)
    for kw in (dict(m=0x1000), dict(v=0x13fc), dict(param=0x3ffc), dict(step=0x1100), dict(step=0x4000), dict(grad=0x1200), dict(grad=0x3004)):
        assert step(_table(**kw)) == -7, kw
    assert step(_table(scales=0x3080), bits=8) == -7                                  # (the 256 codes of m end at 0x3100)
    assert step(_table(), _table()) == -7 and step(_table(), _table(**{**far, 'step': 0x6000})) == -7
    assert step(_table(), _table(**{**far, 'grad': 0x13000})) == -7 and step(_table(n=8192), _table(**far)) == -7
    assert step(_table(), _table(**{**far, 'dtype': 1, 'm': 0x111fc})) == -7          # 256 bfloat16 values end at 0x11200
    long = (2 ** 24 - 1) * 2048
    assert step(_table(n=long + 1)) == -2 and L.igcn_error_string(-7)


def test_the_c_linear_rejects_bad_arguments_before_any_launch():
    L = _lib.lib()
    P = 0x1000

    def linear(x=P, x_dtype=0, ldx=4096, b=P, ldb=4096, sb=P, bias=None, m=4, n=8, k=4096, y=P, dtype=0, ldy=8, ws=P):
        return L.igcn_linear_i8(x, x_dtype, ldx, b, ldb, sb, bias, m, n, k, y, dtype, ldy, ws, None)
    assert linear(dtype=3) == -4 and linear(x_dtype=-1) == -4 and linear(ldx=4095) == -2 and linear(ldb=1) == -2 and linear(ldy=7) == -2 and linear(m=-1) == -2
    assert linear(k=131072, ldx=1 << 18, ldb=1 << 18) == -4 and linear(m=1 << 31) == -2
    for kw in (dict(x=None), dict(b=None), dict(sb=None), dict(y=None), dict(ws=None)):
        assert linear(**kw) == -1, kw
    assert linear(x=0x1002) == -3 and linear(y=0x1002) == -3 and linear(sb=0x1001) == -3 and linear(bias=0x1002) == -3 and linear(ws=0x1008) == -3
    assert linear(m=0, x=None, ws=None) == 0 and linear(n=0, ldy=0, ws=None) == 0
    size = L.igcn_linear_i8_workspace_bytes
    assert size(-1, 4) == -1 and size(4, -1) == -1 and size(4, 131072) == -1 and size(1 << 31, 4) == -1
    assert size(1, 64) == 0 and size(4, 4096) >= 4 * 4096 + 16 and size(3, 8001) >= 3 * 8001 + 12


def test_a_copied_optimizer_keeps_its_settings():
    import copy
    import pickle
    w = torch.nn.Parameter(torch.zeros(4))
    opt = AdamW([w], lr=0.1, state_bits=8, max_grad_norm=2., seed=5)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.max_grad_norm == 2. and other.seed == 5 and other.param_groups[0]['state_bits'] == 8 and other.grad_norm is None


def test_the_c_step_refuses_a_norm_or_a_rate_in_memory_that_it_rewrites():
    L = _lib.lib()

    def step(mx=1., lr_dev=None, ni=None, no=0x9000):
        t = _table()
        return L.igcn_adamw_step(t.buffer_info()[0], 1, 32, 1e-3, lr_dev, 0.9, 0.999, 1e-8, 0.01, mx, ni, no, 0, 0x100, None)
    for at in (0x1000, 0x13fc, 0x3000, 0x4100, 0x6000):                               # parameter, moments, step
        assert step(no=at) == -7 and step(ni=at) == -7 and step(lr_dev=at) == -7 and step(mx=0., lr_dev=at) == -7, hex(at)
    assert step(no=0x2000) == -7                                                      # (a gradient: read by the step, so not to be written)


def _torch_state(w, steps=3):
    """A torch.optim.AdamW state of w after some steps, and the optimizer's groups."""
    opt = torch.optim.AdamW([w], lr=1e-2)
    for k in range(steps):
        w.grad = torch.randn(w.shape, generator=torch.Generator().manual_seed(k)).to(w.dtype)
        opt.step()
    return opt.state_dict()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('transposed,saved_transposed', [(False, False), (True, True), (True, False), (False, True)])
def test_a_loaded_state_has_the_steps_types_and_its_parameters_order(dtype, transposed, saved_transposed):
    """torch.optim.AdamW holds moments in the parameter's type, and a saved tensor may lie in memory in another order: what is loaded are float32
    moments, laid out like the parameter, of the same values."""
    def param(tr):
        data = torch.randn(6, 10, generator=torch.Generator().manual_seed(9)).to(dtype)
        return torch.nn.Parameter(data.t().contiguous().t() if tr else data)
    saved = _torch_state(param(saved_transposed))
    w = param(transposed)
    opt = AdamW([w], lr=1e-2)
    opt.load_state_dict(saved)
    for name in ('exp_avg', 'exp_avg_sq'):
        got, want = opt.state[w][name], saved['state'][0][name]
        assert want.dtype == dtype and got.dtype == torch.float32 and torch.equal(got, want.float()), name
        assert ops._same_order(w, got) and got.data_ptr() != want.data_ptr(), name
    assert opt.state[w]['step'].dtype == torch.float32 and float(opt.state[w]['step']) == 3. and opt.param_groups[0]['state_bits'] == 32


def test_a_state_that_does_not_fit_is_refused_and_changes_nothing():
    """8-bit codes share scales in memory order, so they do not go to a parameter of another order; nor does a moment of another shape, nor half a
    form.  The optimizer stays as it was."""
    w = torch.nn.Parameter(torch.zeros(16, 24))
    tr = torch.nn.Parameter(torch.zeros(24, 16).t())

    def state(p, **new):
        codes = [torch.full_like(p, 5, dtype=torch.uint8).view(d) for d in ops.MOMENT_DTYPES]
        s = {'step': torch.tensor(4.), 'exp_avg': codes[0].detach(), 'exp_avg_sq': codes[1].detach(), 'scales': torch.rand(3, 2)}
        s.update(new)
        opt = AdamW([p], lr=0.5, state_bits=8)
        return {'state': {0: {k: v for k, v in s.items() if v is not None}}, 'param_groups': opt.state_dict()['param_groups']}
    fine = AdamW([w], lr=1e-2)
    fine.load_state_dict(state(w))
    assert fine.state[w]['exp_avg'].dtype == torch.float8_e4m3fn and fine.param_groups[0]['state_bits'] == 8 and fine.param_groups[0]['lr'] == 0.5
    assert torch.equal(fine.state[w]['exp_avg'].view(torch.uint8), torch.full((16, 24), 5, dtype=torch.uint8))
    f32 = torch.zeros(16, 24)
    bad = [(w, state(tr)), (tr, state(w)), (w, state(w, scales=torch.rand(4, 2))), (w, state(w, exp_avg=f32)), (w, state(w, exp_avg_sq=None)),
           (w, state(w, scales=None)), (w, state(w, exp_avg=f32, exp_avg_sq=torch.zeros(24, 16), scales=None)), (w, state(w, step=None)),
           (w, state(w, step=torch.zeros(2))), (w, state(w, exp_avg=f32[:8], exp_avg_sq=f32[:8], scales=None))]
    for i, (p, saved) in enumerate(bad):
        opt = AdamW([p], lr=1e-2, state_bits=32)
        opt.state[p].update(step=torch.tensor(1.), exp_avg=torch.zeros_like(p).detach(), exp_avg_sq=torch.zeros_like(p).detach())
        held = dict(opt.state[p])
        with pytest.raises(ValueError):
            opt.load_state_dict(saved)
            print('not refused:', i)
        assert opt.param_groups[0]['lr'] == 1e-2 and opt.param_groups[0]['state_bits'] == 32 and all(opt.state[p][k] is v for k, v in held.items()), i
    a, b = torch.nn.Parameter(torch.zeros(16, 24)), torch.nn.Parameter(torch.zeros(16, 24))
    mixed = state(w)
    mixed['param_groups'][0]['params'] = [0, 1]
    mixed['state'][1] = {'step': torch.tensor(4.), 'exp_avg': f32, 'exp_avg_sq': f32}
    opt = AdamW([a, b], lr=1e-2)
    with pytest.raises(ValueError):
        opt.load_state_dict(mixed)
    assert opt.param_groups[0]['lr'] == 1e-2 and not opt.state


@pytest.mark.parametrize('make', [lambda ps: AdamW(ps, lr=0.1), lambda ps: AdamW(ps, lr=0.1, state_bits=8), lambda ps: torch.optim.Adam(ps, lr=0.1),
                                  lambda ps: torch.optim.SGD(ps, lr=0.1, momentum=0.9)])
def test_a_captured_steps_key_names_the_memory_the_optimizer_writes(make):
    """A captured step holds the addresses of the parameters and of the optimizer's state: whatever replaces one of them — load_state_dict, a new
    .data — makes another key; a step, which rewrites them in place, does not."""
    import copy
    from igcn_cf_amd.trainer import BPRTrainer
    ps = [torch.nn.Parameter(torch.zeros(300, 4)), torch.nn.Parameter(torch.zeros(7))]
    trainer = BPRTrainer.__new__(BPRTrainer)
    trainer.model, trainer.opt, trainer.batch_size = torch.nn.Module(), make(ps), 4
    for p in ps:
        p.grad = torch.ones_like(p)
        if isinstance(trainer.opt, AdamW):
            trainer.opt._state_of(p, trainer.opt.param_groups[0]['state_bits'])
    if not isinstance(trainer.opt, AdamW):
        trainer.opt.step()
    key = trainer._graph_key()
    held = [dict(trainer.opt.state[p]) for p in ps]                                   # (so that no address comes back)
    if not isinstance(trainer.opt, AdamW):
        trainer.opt.step()
    assert trainer._graph_key() == key
    trainer.opt.load_state_dict(copy.deepcopy(trainer.opt.state_dict()))
    after = trainer._graph_key()
    assert after != key and trainer._graph_key() == after
    old, ps[1].data = ps[1].data, torch.zeros(7)
    assert trainer._graph_key() != after and held and old is not None
    if isinstance(trainer.opt, AdamW):
        trainer.opt.state.clear()
        assert trainer._graph_key() != after


def test_the_gpu_tests_reach_every_kernel_of_the_8_bit_product(tmp_path):
    """The rule that chooses among them (csrc/gemm_i8_rule.h, plain C++) is compiled here and asked about every size of the GPU tests: each kernel has to
    come up in each of its forms — tiles from rows on and off 16-byte multiples, streams of rows on and off 4-byte ones, rows of fewer than 16 codes."""
    import os
    import re
    import subprocess
    from tests import test_i8_gpu as G
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'igcn_cf_amd', 'csrc')
    names = re.search(r'enum class I8Way \{(.*?)\};', open(os.path.join(csrc, 'gemm_i8_rule.h')).read(), re.S).group(1)
    names = re.findall(r'\bk\w+', re.sub(r'//.*', '', names))
    (tmp_path / 'ask.cpp').write_text('''
#include "gemm_i8_rule.h"
#include <cstdio>
using namespace igcn;
int main()
{
    long long m, n, k, lda, ldb, at;
    int f32;
    while (scanf("%lld %lld %lld %lld %lld %lld %d", &m, &n, &k, &lda, &ldb, &at, &f32) == 7)
        printf("%d %d %d %d %d %d\\n", (int)i8_way(m, n, k, lda, ldb, f32), i8_direct(at, at, lda, ldb, k), i8_any_byte(at, lda) || i8_any_byte(at, ldb),
               i8_quantises_on_the_way(m, n, k), i8_shares_depth(n),
               i8_asks_ahead(m, n, k, f32));
}
''')
    subprocess.run(['g++', '-std=c++17', '-O1', '-Wall', '-Werror', '-I', csrc, str(tmp_path / 'ask.cpp'), '-o', str(tmp_path / 'ask')], check=True)

    def ask(rows):
        got = subprocess.run([str(tmp_path / 'ask')], input='\n'.join(' '.join(map(str, r)) for r in rows), check=True, stdout=subprocess.PIPE, text=True).stdout
        return [[int(x) for x in line.split()] for line in got.splitlines()]
    sizes = [s for s in G.SIZES + G.TILE_SIZES if min(s) > 0]
    rows = [(m, n, k, k, k, 0, f32) for m, n, k in sizes for f32 in (0, 1)]
    rows += [(300, 700, k, 2200 * step, 2230 * step, off, f32) for off in (0, 1) for k in (1, 15, 64, 380, 2100) for step in (1, 3) for f32 in (0, 1)]
    rows += [(m, n, 100, lda or 100, ldb or 100, 0, 1) for m, n, lda, ldb in G.APART_SIZES]
    met, ahead = set(), set()
    for (m, n, k, *_), (way, direct, byte, _, _, asks) in zip(rows, ask(rows)):
        name = names[way]
        ahead |= {(name, asks)} if direct else set()
        met.add((name, 'short') if k < 16 else (name, direct) if 'Tiles' in name and 'Stream' not in name else (name, byte))
    want = {(name, form) for name in names for form in (0, 1)}
    assert len(names) == 10 and want <= met, sorted(want - met)
    assert {name for name, form in met if form == 'short'} >= {'kStream', 'kStreamTwoGroups', 'kTiles64x128', 'kTiles128', 'kTiles64'}
    assert ahead >= {(name, asks) for name in ('kTiles64x128', 'kTiles128', 'kTiles64') for asks in (0, 1)}
    few = [(m, n, k, k, k + past, 0, 1) for m, n, k, _, past in G.FEW_SIZES]
    met = {(shares, byte, k < 16, dtype) for (m, n, k, dtype, _), (_, _, byte, fused, shares, _) in zip(G.FEW_SIZES, ask(few)) if fused}
    assert {(s, b, t) for s, b, _, t in met} == {(s, b, t) for s in (0, 1) for b in (0, 1) for t in G.DTYPES} and {s for s, _, short, _ in met if short} == {0, 1}


def test_a_trainer_takes_the_sum_over_ranks_of_shares_only():
    """A model's all_reduce is the clipped norm's where its parameters are marked as shares (dist's models mark them), not where every rank has all of
    them and the method means something else; a slice_reduce_fn that is replaced later is followed."""
    from igcn_cf_amd.trainer import BPRTrainer
    trainer = BPRTrainer.__new__(BPRTrainer)
    trainer.model = torch.nn.Linear(3, 3)
    trainer.model.all_reduce = lambda t: t
    trainer.config = {'optimizer': 'AdamW', 'lr': 0.1, 'max_grad_norm': 1.}
    trainer.initialize_optimizer()
    assert trainer.opt.norm_reduce_fn is None
    for p in trainer.model.parameters():
        p.is_share = True
    trainer.initialize_optimizer()
    assert trainer.opt.norm_reduce_fn is trainer.model.all_reduce
    trainer.opt.step = lambda: None
    trainer.model.slice_reduce_fn = lambda t: t
    trainer._optimizer_step()
    assert trainer.opt.norm_reduce_fn is trainer.model.slice_reduce_fn
