"""Rows in 8-bit integers (ops.quantize_rows_i8 / dequantize_rows_i8) and their product (ops.matmul_i8 / linear_i8) on the GPU: codes
and sums are exact, so codes are compared one by one and scores to the few float32 roundings behind the sum."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _codes(shape, g, lo=-128):
    return torch.randint(lo, 128, shape, device=DEV, generator=g, dtype=torch.int8)


def _quantized(x):
    """(codes, scales) from float64: the quotient of two float32 numbers, rounded to 64 bits, is never on the wrong side of a half."""
    x = x.double()
    s = (x.abs().amax(1) / 127).float() if x.shape[1] else torch.zeros(x.shape[0], device=x.device)
    q = torch.round(x / torch.where(s > 0, s, 1.).double()[:, None]) * (s > 0)[:, None]
    return q.clamp(-127, 127).to(torch.int8), s


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,k', [(1, 1), (3, 7), (5, 16), (64, 63), (65, 64), (1000, 64), (9, 65), (130, 128), (7, 255), (17, 256), (4, 1000),
                                    (3, 1024), (2, 2049), (3, 8191), (2, 8192), (1, 70001), (0, 5), (4, 0)])
def test_codes_and_scales_are_the_nearest(rows, k, dtype):
    from igcn_cf_amd import ops
    g = _rng(rows * 1000 + k)
    x = (torch.randn(rows, k, device=DEV, generator=g) * torch.exp(2 * torch.randn(rows, 1, device=DEV, generator=g))).to(dtype)
    if rows > 2 and k:
        x[1] = 0                                                                       # a row of zeros
        x[2] = x[2].abs().amax() * torch.arange(k, device=DEV).remainder(3).sub(1).to(dtype)      # -max, 0, max
    q, s = ops.quantize_rows_i8(x)
    want_q, want_s = _quantized(x)
    assert q.dtype == torch.int8 and torch.equal(s, want_s) and torch.equal(q, want_q)
    for out in DTYPES:
        y = ops.dequantize_rows_i8(q, s, dtype=out)
        assert y.dtype == out and torch.equal(y, (q.float() * s[:, None]).to(out))


def test_ties_go_to_the_even_code_and_small_rows_keep_their_size():
    """max 254 makes the scale exactly 2: odd values are halves.  Rows of the smallest magnitudes have scales of few digits (or 0, where
    max / 127 is below float32): codes stay the nearest within -127 ... 127."""
    from igcn_cf_amd import ops
    x = torch.arange(-254., 255., device=DEV)[None, :]
    q, s = ops.quantize_rows_i8(x)
    assert float(s) == 2. and torch.equal(q[0].long(), torch.round(x[0] / 2).long())
    for scale in (1e-30, 1e-37, 1e-38, 1e-40, 1e-42, 1e-44, 3e38):
        x = (torch.linspace(-1, 1, 301, dtype=torch.float64, device=DEV) * scale).float()[None, :]
        q, s = ops.quantize_rows_i8(x)
        want_q, want_s = _quantized(x)
        assert torch.equal(s, want_s) and torch.equal(q, want_q), scale


def test_broken_rows_show_and_leave_the_others_alone():
    from igcn_cf_amd import ops
    x = torch.randn(6, 200, device=DEV, generator=_rng(1))
    clean_q, clean_s = ops.quantize_rows_i8(x)
    x[1, 150], x[3, 0], x[4, 199] = float('nan'), float('inf'), -float('inf')
    q, s = ops.quantize_rows_i8(x)
    assert torch.isnan(s).tolist() == [False, True, False, True, True, False] and not q[1].any() and not q[3:5].any()
    for r in (0, 2, 5):
        assert torch.equal(q[r], clean_q[r]) and s[r] == clean_s[r]
    y = ops.linear_i8(x, clean_q, clean_s)
    assert torch.isnan(y).all(1).tolist() == [False, True, False, True, True, False]


def test_rows_apart_and_off_alignment():
    """Leading dimensions other than the width, every second row, and rows that start at any byte."""
    from igcn_cf_amd import ops
    g = _rng(2)
    for dtype in DTYPES:
        big = torch.randn(50, 300, device=DEV, generator=g).to(dtype)
        for x in (big[:, 3:260], big[::2, :64], big[1:, 1:130], big[7:8, 5:6]):
            q, s = ops.quantize_rows_i8(x)
            want_q, want_s = _quantized(x)
            assert torch.equal(q, want_q) and torch.equal(s, want_s)
    ca, cb = _codes((200, 400), g), _codes((300, 500), g)
    sa, sb = torch.rand(200, device=DEV, generator=g), torch.rand(300, device=DEV, generator=g)
    for off in (0, 1, 2, 3, 4, 8, 15):
        for k in (1, 15, 16, 31, 64, 100, 129, 256, 380):
            for step in (1, 3):
                a, b = ca[::step, off:off + k], cb[off % 3::step, 2 * off:2 * off + k]
                check(a, sa[:a.shape[0]], b, sb[:b.shape[0]])
    y = ops.dequantize_rows_i8(ca[::3, 5:77], sa[:67])
    assert torch.equal(y, ca[::3, 5:77].float() * sa[:67, None])


def check(a, sa, b, sb, bias=None, dtype=torch.float32):
    """matmul_i8 against 64 bits: the sum is exact, then it is rounded to float32, multiplied twice, and the bias added: 3 roundings of the
    product and one of the result, and the output type's own."""
    from igcn_cf_amd import ops
    y = ops.matmul_i8(a, sa, b, sb, bias=bias, dtype=dtype)
    assert y.dtype == dtype and y.shape == (a.shape[0], b.shape[0])
    prod = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    want = prod if bias is None else prod + bias.double()
    off = 3 * U * prod.abs() + U * want.abs()
    half = 0. if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    off = off + half * (want.abs() + off) + (2.0 ** -25 if dtype == torch.float16 else 0.)
    top = torch.finfo(dtype).max
    want = torch.where(want.abs() > top, torch.sign(want) * float('inf'), want) if dtype == torch.float16 else want
    same = torch.isinf(want) & (y.double() == want)
    bad = ~(((y.double() - want).abs() <= off * (1 + 1e-6) + 1e-45) | same)
    assert not bool(bad.any()), (tuple(a.shape), tuple(b.shape), dtype, int(bad.sum()), bad.nonzero()[:4].tolist())
    return y


SIZES = [(1, 1, 1), (1, 17, 64), (2, 33, 16), (3, 5, 48), (4, 100, 8), (5, 1000, 64), (8, 64, 1024), (13, 77, 129), (16, 129, 100), (17, 300, 64), (31, 31, 31),
         (32, 200, 4096), (33, 65, 63), (48, 96, 256), (63, 1025, 64), (64, 64, 64), (65, 129, 100), (100, 4097, 128), (127, 127, 255), (128, 256, 512), (129, 257, 65),
         (255, 255, 1000), (256, 512, 192), (257, 300, 515), (300, 700, 2048), (512, 512, 4096), (513, 1029, 333), (1, 5000, 8191), (7, 3001, 5000), (1000, 1, 777),
         (7, 5001, 2100), (16, 8000, 2049), (12, 4100, 4096), (3, 30000, 333), (2, 25000, 64), (30, 4096, 2000), (22, 1000, 130), (1800, 2050, 2064), (1800, 2050, 2051),
         (189, 48, 5391), (97, 66, 4678), (250, 500, 1999), (64, 2048, 77), (5000, 17, 40), (2100, 2100, 160), (2100, 2100, 71), (0, 5, 3), (5, 0, 3), (6, 7, 0)]


@pytest.mark.parametrize('m,n,k', SIZES)
def test_products_of_all_sizes(m, n, k):
    g = _rng(m * 31 + n * 7 + k)
    a, b = _codes((m, k), g), _codes((n, k), g)
    sa, sb = torch.exp(torch.randn(m, device=DEV, generator=g) - 5), torch.exp(torch.randn(n, device=DEV, generator=g) - 5)
    bias = torch.randn(n, device=DEV, generator=g)
    for dtype in DTYPES:
        check(a, sa, b, sb, None, dtype)
        check(a, sa, b, sb, bias, dtype)


def test_the_longest_sums_and_the_largest_codes():
    """131 071 products of -128 * -128 are 2 147 467 264 < 2^31; and sums past 2^24 are rounded once."""
    from igcn_cf_amd import ops
    for k in (131071, 65536, 40000):
        for m in (1, 3, 40):
            a = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
            b = torch.full((70, k), -128, dtype=torch.int8, device=DEV)
            b[1::2] = 127
            one = torch.ones(70, device=DEV)
            y = check(a, one[:m], b, one)
            assert float(y[0, 0]) == np.float32(k * 16384) and float(y[0, 1]) == np.float32(-k * 128 * 127)
    with pytest.raises(ops._lib.IgcnError):
        ops.matmul_i8(torch.zeros(1, 131072, dtype=torch.int8, device=DEV), torch.ones(1, device=DEV), torch.zeros(1, 131072, dtype=torch.int8, device=DEV), torch.ones(1, device=DEV))


@pytest.mark.parametrize('m', [1, 3, 40])
def test_offsets_past_32_bits(m):
    """Rows behind the 2^31st byte of b, and outputs behind the 2^32nd byte of y."""
    g = _rng(3)
    k, n = 8192, 270000                                                                 # 2.2 GB of codes
    a, b = _codes((m, k), g), torch.empty((n, k), dtype=torch.int8, device=DEV)
    for r in range(0, n, 30000):
        b[r:r + 30000] = _codes((30000, k), g)
    sa, sb = torch.rand(m, device=DEV, generator=g), torch.rand(n, device=DEV, generator=g)
    from igcn_cf_amd import ops
    y = ops.matmul_i8(a, sa, b, sb)
    at = torch.cat([torch.arange(100, device=DEV), torch.arange(n - 9000, n, device=DEV)])
    want = (a.double() @ b[at].double().t()) * sa.double()[:, None] * sb[at].double()
    assert bool(((y[:, at].double() - want).abs() <= 4 * U * want.abs() * (1 + 1e-6)).all())
    if m == 40:
        del y, b
        m, n, k = 40000, 30000, 16                                                      # 4.8 GB of scores
        a, b = _codes((m, k), g), _codes((n, k), g)
        sa, sb = torch.rand(m, device=DEV, generator=g), torch.rand(n, device=DEV, generator=g)
        y = ops.matmul_i8(a, sa, b, sb)
        for rows in (slice(0, 64), slice(m - 64, m), slice(17890, 17900)):
            want = (a[rows].double() @ b.double().t()) * sa[rows].double()[:, None] * sb.double()
            assert bool(((y[rows].double() - want).abs() <= 4 * U * want.abs() * (1 + 1e-6)).all())


@pytest.mark.parametrize('m,n,k,dtype', [(1, 1000, 64, torch.float32), (1, 700, 4096, torch.bfloat16), (4, 333, 8192, torch.float16), (16, 500, 100, torch.float32),
                                         (20, 500, 1000, torch.bfloat16), (300, 400, 64, torch.float32), (2, 99, 131071, torch.float32), (3, 50, 7, torch.bfloat16), (2, 600001, 40, torch.float32),
                                         (8, 40000, 500, torch.bfloat16), (4, 16384, 1000, torch.float16), (4, 16385, 1000, torch.float16), (1, 33000, 15, torch.float32)])
def test_a_linear_is_its_two_parts_and_takes_the_inputs_type(m, n, k, dtype):
    from igcn_cf_amd import ops
    g = _rng(k)
    x = torch.randn(m, k, device=DEV, generator=g).to(dtype)
    b, sb = _codes((n, k), g), torch.rand(n, device=DEV, generator=g)
    bias = torch.randn(n, device=DEV, generator=g)
    q, s = _quantized(x)
    for out in (None, *DTYPES):
        y = ops.linear_i8(x, b, sb, bias=bias, dtype=out)
        assert y.dtype == (out or dtype)
        assert torch.equal(y, ops.matmul_i8(q, s, b, sb, bias=bias, dtype=out or dtype))
    x[-1, -1] = float('nan')
    if m > 1:
        x[0] = 0
    y = ops.linear_i8(x, b, sb, bias=bias)
    assert bool(torch.isnan(y[-1]).all()) and (m == 1 or torch.equal(y[0], bias.to(dtype)))


def test_captured_products_follow_new_inputs_and_streams_do_not_meet():
    """One captured call replayed on changed inputs, twice captured calls replayed in turn, and eager calls on several streams at once."""
    from igcn_cf_amd import ops
    g = _rng(9)
    for m, n, k in ((1, 2000, 4096), (4, 1000, 8192), (70, 300, 500), (300, 600, 256)):
        x, b = torch.randn(m, k, device=DEV, generator=g), _codes((n, k), g)
        sb = torch.rand(n, device=DEV, generator=g)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.linear_i8(x, b, sb)
        torch.cuda.current_stream().wait_stream(side)
        graphs, outs = [], []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(ops.linear_i8(x, b, sb))
            graphs.append(graph)
        for rep in range(4):
            x.copy_(torch.randn(m, k, device=DEV, generator=g))
            want = ops.linear_i8(x, b, sb)
            torch.cuda.synchronize()
            for graph, out in zip(graphs, outs):
                out.zero_()
                graph.replay()
            torch.cuda.synchronize()
            for out in outs:
                assert torch.equal(out, want)
        streams, got = [torch.cuda.Stream() for _ in range(4)], []
        torch.cuda.synchronize()
        for s in streams:
            with torch.cuda.stream(s):
                got.append([ops.linear_i8(x, b, sb) for _ in range(3)])
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for ys in got for y in ys)


@pytest.mark.parametrize('m,n', [(5, 40), (20, 9), (150, 70)])
def test_rows_megabytes_apart(m, n):
    """Leading dimensions over 2^23: offsets within a tile would pass 31 bits."""
    from igcn_cf_amd import ops
    g, k, ld = _rng(m), 100, (1 << 23) + 48
    a, b = _codes((m, k), g), _codes((n, k), g)
    sa, sb = torch.rand(m, device=DEV, generator=g), torch.rand(n, device=DEV, generator=g)
    for far_a, far_b in ((True, False), (False, True), (True, True)):
        def spread(t, far):
            if not far:
                return t
            rows = torch.empty((t.shape[0] - 1) * ld + k, dtype=torch.int8, device=DEV).as_strided(t.shape, (ld, 1))
            return rows.copy_(t)
        y = check(spread(a, far_a), sa, spread(b, far_b), sb)
        assert torch.equal(y, ops.matmul_i8(a, sa, b, sb))


def test_more_rows_and_columns_than_a_launch_takes():
    """2^22 rows and 2^23 columns are what one launch is given."""
    from igcn_cf_amd import ops
    g = _rng(5)
    x = torch.randn((1 << 22) + 70, 3, device=DEV, generator=g).to(torch.bfloat16)
    q, s = ops.quantize_rows_i8(x)
    want_q, want_s = _quantized(x)
    assert torch.equal(q, want_q) and torch.equal(s, want_s)
    assert torch.equal(ops.dequantize_rows_i8(q, s), q.float() * s[:, None])
    q, s = _codes((2, (1 << 23) + 11), g), torch.rand(2, device=DEV, generator=g)
    assert torch.equal(ops.dequantize_rows_i8(q, s, dtype=torch.float16), (q.float() * s[:, None]).half())


def test_refusals():
    from igcn_cf_amd import ops
    Error = ops._lib.IgcnError
    x, q, s = torch.zeros(6, 32, device=DEV), torch.zeros(6, 32, dtype=torch.int8, device=DEV), torch.ones(6, device=DEV)
    bad = [lambda: ops.quantize_rows_i8(x.double()), lambda: ops.quantize_rows_i8(x[0]), lambda: ops.quantize_rows_i8(x.t()), lambda: ops.quantize_rows_i8(x[:1].expand(6, 32)),
           lambda: ops.quantize_rows_i8(x[None]), lambda: ops.quantize_rows_i8(x[:, ::2]), lambda: ops.quantize_rows_i8(x.to_sparse()), lambda: ops.quantize_rows_i8([1.]),
           lambda: ops.dequantize_rows_i8(x, s), lambda: ops.dequantize_rows_i8(q, s[:5]), lambda: ops.dequantize_rows_i8(q, s.double()), lambda: ops.dequantize_rows_i8(q, s.cpu()),
           lambda: ops.dequantize_rows_i8(q, s, dtype=torch.float64), lambda: ops.dequantize_rows_i8(q.view(torch.uint8), s)]
    for name, call in (('a', ops.matmul_i8), ('x', ops.linear_i8)):
        def product(a=None, sa=s, b=q, sb=s, call=call, own=q if name == 'a' else x, **kw):
            a = own if a is None else a
            return call(a, sa, b, sb, **kw) if call is ops.matmul_i8 else call(a, b, sb, **kw)
        assert product().shape == (6, 6)
        own = q if name == 'a' else x
        bad += [lambda f=product: f(b=q[:, :31]), lambda f=product: f(sb=s[:5]), lambda f=product: f(sb=s[None]), lambda f=product: f(b=x), lambda f=product: f(b=q.t()),
                lambda f=product: f(bias=s[:3]), lambda f=product: f(bias=s.half()), lambda f=product: f(bias=s.cpu()), lambda f=product: f(b=q.cpu()),
                lambda f=product: f(dtype=torch.int32), lambda f=product, o=own: f(a=o[:, :, None]), lambda f=product, o=own: f(a=o.cpu()),
                lambda f=product, o=own: f(a=o[:, ::2]), lambda f=product, o=own: f(a=o.double())]
    bad += [lambda: ops.matmul_i8(q, s[:5], q, s), lambda: ops.matmul_i8(x, s, q, s), lambda: ops.linear_i8(q, q, s)]
    for i, call in enumerate(bad):
        with pytest.raises(Error):
            call()
            print('not refused:', i)


def test_quantised_values_past_32_bits():
    from igcn_cf_amd import ops
    rows, k = 40000, 60000                                                               # 2.4e9 values, 4.8 GB
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEV)
    x[-40:] = torch.randn(40, k, device=DEV, generator=_rng(8)).to(torch.bfloat16)
    q, s = ops.quantize_rows_i8(x)
    want_q, want_s = _quantized(x[-40:])
    assert torch.equal(q[-40:], want_q) and torch.equal(s[-40:], want_s) and not bool(s[:-40].any()) and not bool(q[-80:-40].any())
    y = ops.dequantize_rows_i8(q, s, dtype=torch.float16)
    assert torch.equal(y[-40:], (want_q.float() * want_s[:, None]).half()) and not bool(y[-80:-40].any())


# Sizes at which the rule of csrc/gemm_i8_rule.h goes to its larger kernels (test_operators_cpu asks it whether every one is met): partial last tiles and
# stages, rows on and off 16-byte multiples.
TILE_SIZES = [(3600, 3600, 272), (3600, 3600, 259), (4000, 3400, 131), (513, 1029, 999), (27, 20956, 1381), (300, 700, 2051), (64, 4096, 2053), (300, 700, 2049),
              (65, 8200, 2064), (2000, 2000, 4099), (700, 4200, 333), (1030, 3300, 1040), (100, 30000, 48), (70, 40000, 13), (9, 30000, 7), (40, 30000, 15), (40, 12000, 2500), (64, 1200, 9), (128, 96421, 64),
              (300, 60001, 112), (33, 530001, 16)]


@pytest.mark.parametrize('m,n,k', TILE_SIZES)
def test_products_in_the_larger_tiles(m, n, k):
    g = _rng(m * 31 + n * 7 + k)
    a, b = _codes((m, k), g), _codes((n, k), g)
    sa, sb = torch.exp(torch.randn(m, device=DEV, generator=g) - 5), torch.exp(torch.randn(n, device=DEV, generator=g) - 5)
    bias = torch.randn(n, device=DEV, generator=g)
    for dtype in (torch.float32, torch.bfloat16):
        check(a, sa, b, sb, bias if dtype == torch.bfloat16 else None, dtype)


def test_rows_of_tiles_apart_and_off_alignment():
    """As test_rows_apart_and_off_alignment, at sizes that go through LDS: rows that start at any byte, every third row, a depth of one stage, of several and
    of a few codes."""
    g = _rng(21)
    ca, cb = _codes((900, 2200), g), _codes((2110, 2230), g)
    sa, sb = torch.rand(900, device=DEV, generator=g), torch.rand(2110, device=DEV, generator=g)
    for off in (0, 1, 2, 3, 4, 8, 15):
        for k in (1, 15, 16, 31, 64, 100, 129, 256, 380, 600, 2100):
            for step in (1, 3):
                a, b = ca[:300 * step:step, off:off + k], cb[off % 3:off % 3 + 700 * step:step, 2 * off:2 * off + k]
                check(a, sa[:300], b, sb[:700], dtype=torch.bfloat16 if off % 2 else torch.float32)


APART_SIZES = [(150, 2000, (1 << 23) + 48, None), (150, 2000, (1 << 23) + 49, None), (2000, 150, None, (1 << 23) + 48), (2000, 150, None, (1 << 23) + 51)]


@pytest.mark.parametrize('m,n,lda,ldb', APART_SIZES)
def test_more_rows_megabytes_apart_than_stream(m, n, lda, ldb):
    """Leading dimensions over 2^23 where the size asks for tiles: offsets within one would pass 31 bits."""
    from igcn_cf_amd import ops
    g, k = _rng(m), 100
    a, b = _codes((m, k), g), _codes((n, k), g)
    sa, sb = torch.rand(m, device=DEV, generator=g), torch.rand(n, device=DEV, generator=g)

    def spread(t, ld):
        if ld is None:
            return t
        rows = torch.empty((t.shape[0] - 1) * ld + k, dtype=torch.int8, device=DEV).as_strided(t.shape, (ld, 1))
        return rows.copy_(t)
    y = check(spread(a, lda), sa, spread(b, ldb), sb)
    assert torch.equal(y, ops.matmul_i8(a, sa, b, sb))


def test_more_rows_than_a_launch_against_two_megabytes_apart():
    """65535 x 32 rows of a are what one launch is given there."""
    g, m, k, ld = _rng(23), 65535 * 32 + 2900, 16, (1 << 23) + 16
    a, b = _codes((m, k), g), torch.empty(ld + k, dtype=torch.int8, device=DEV).as_strided((2, k), (ld, 1))
    b.copy_(_codes((2, k), g))
    sa, sb = torch.rand(m, device=DEV, generator=g), torch.rand(2, device=DEV, generator=g)
    check(a, sa, b, sb, dtype=torch.float16)


# (m, n, k, type of x, bytes between rows of b past k): the products that quantise on their way, each kernel of them
FEW_SIZES = [(m, n, k, dtype, past) for dtype in DTYPES for m, n, k, past in
             ((1, 33, 64, 0), (3, 1000, 130, 0), (8, 500, 77, 0), (2, 1024, 12, 2), (5, 40001, 64, 0), (8, 33000, 200, 1), (1, 50000, 13, 0), (7, 70000, 9, 3))]


@pytest.mark.parametrize('m,n,k,dtype,past', FEW_SIZES)
def test_a_few_short_rows_of_every_type(m, n, k, dtype, past):
    from igcn_cf_amd import ops
    g = _rng(m + n + k)
    x = torch.randn(m, k, device=DEV, generator=g).to(dtype)
    b, sb = _codes((n, k + past), g)[:, :k], torch.rand(n, device=DEV, generator=g)
    q, s = _quantized(x)
    assert torch.equal(ops.linear_i8(x, b, sb, dtype=torch.float32), check(q, s, b, sb))
