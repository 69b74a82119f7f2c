"""The cases the optimizer step and the 8-bit scoring operators are measured on, with the operators' plain forms.

An AdamW step over many tensors (moments in 32 bits or in 8, the gradient norm over all of them and clipping by it), rows quantised
to 8-bit integers, and the product of such rows with a scale for each row of either side."""
import math

import torch

own = False

DEVICE = 'cuda'
BLOCK = 128                      # elements that share a scale in the 8-bit moments
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2
MAX_NORM = 1.0
SEED = 2021
STEP = 10                        # steps taken before the measured one
DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
LARGEST = 1 << 27                # elements of the largest tables and score blocks
LARGEST_PRODUCT = 8192 * 8192 * 4096


# ---- cases ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the two tables of a toy split, every step of its training: latency counts
        {'name': 'adamw_small_tables', 'op': 'adamw', 'bits': 32, 'tensors': 2, 'rows': 300, 'width': 64, 'dtype': 'float32', 'clip': False},
        # the embedding table of LightGCN on the Amazon-like split, one step
        {'name': 'adamw_amazon_table', 'op': 'adamw', 'bits': 32, 'tensors': 1, 'rows': 206151, 'width': 64, 'dtype': 'float32', 'clip': False},
        # the weights of a bfloat16 model in several layers, odd sizes among them, clipped by their common norm
        {'name': 'adamw_layers_bf16_clip', 'op': 'adamw', 'bits': 32, 'tensors': 15, 'rows': 4099, 'width': 1024, 'dtype': 'bfloat16', 'clip': True},
        # the same toy tables with moments in 8 bits
        {'name': 'adamw8_small_tables', 'op': 'adamw', 'bits': 8, 'tensors': 2, 'rows': 300, 'width': 64, 'dtype': 'float32', 'clip': False},
        # the Amazon-like table with moments in 8 bits, clipped
        {'name': 'adamw8_amazon_table_clip', 'op': 'adamw', 'bits': 8, 'tensors': 1, 'rows': 206151, 'width': 64, 'dtype': 'float32', 'clip': True},
        # a rank's share of the tables too large for one: what 8-bit moments are for
        {'name': 'adamw8_large_table', 'op': 'adamw', 'bits': 8, 'tensors': 1, 'rows': 1000003, 'width': 128, 'dtype': 'float32', 'clip': False},
        # the item and user rows of the Amazon-like split made 8-bit once after training, and the values they stand for
        {'name': 'quantize_amazon_table', 'op': 'quantize', 'rows': 206151, 'width': 64, 'dtype': 'float32'},
        # a chunk of wide bfloat16 activations, odd width
        {'name': 'quantize_wide_bf16', 'op': 'quantize', 'rows': 2048, 'width': 8191, 'dtype': 'bfloat16'},
        # one user asks: its fp32 row against all 8-bit item rows of the Amazon-like split
        {'name': 'linear_one_user', 'op': 'linear', 'm': 1, 'n': 96421, 'k': 64, 'dtype': 'float32', 'out': 'float32', 'bias': False},
        # a test batch of 512 users against the same items
        {'name': 'matmul_512_users', 'op': 'matmul', 'm': 512, 'n': 96421, 'k': 64, 'out': 'float32', 'bias': False},
        # a few rows through a wide layer: one step of serving
        {'name': 'linear_wide_4_rows', 'op': 'linear', 'm': 4, 'n': 16384, 'k': 8192, 'dtype': 'bfloat16', 'out': 'bfloat16', 'bias': True},
        # a long chunk of rows through a wide layer: the matrix cores' case, and the largest
        {'name': 'matmul_large', 'op': 'matmul', 'm': 8192, 'n': 8192, 'k': 4096, 'out': 'bfloat16', 'bias': True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['adamw', 'adamw', 'quantize', 'linear', 'matmul'])
    dtype = rng.choice(['float32', 'bfloat16', 'float16'])
    if op == 'adamw':
        tensors, width = rng.randint(1, 15), _log(rng, 1, 2048)
        rows = _log(rng, 1, max(2, min(1 << 20, LARGEST // 2 // (tensors * width))))
        return {'op': op, 'bits': rng.choice([8, 32]), 'tensors': tensors, 'rows': rows, 'width': width, 'dtype': dtype, 'clip': rng.random() < 0.5}
    if op == 'quantize':
        width = _log(rng, 1, 8192)
        return {'op': op, 'rows': _log(rng, 1, max(2, min(1 << 18, (1 << 25) // width))), 'width': width, 'dtype': dtype}
    m, k = _log(rng, 1, 8192 if op == 'matmul' else 64), _log(rng, 16, 8192)
    n = _log(rng, 16, max(17, min(131072, LARGEST_PRODUCT // (m * k), LARGEST // 2 // m, LARGEST // k)))
    case = {'op': op, 'm': m, 'n': n, 'k': k, 'out': rng.choice(['float32', 'bfloat16', 'float16']), 'bias': rng.random() < 0.5}
    return dict(case, dtype=dtype) if op == 'linear' else case


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def _shapes(case):
    """Tables first; from the third tensor on also vectors and odd blocks, as the layers of a model have them."""
    rows, width = case['rows'], case['width']
    kinds = [(rows, width), (max(1, rows // 2), width), (width,), (rows // 3 + 1, width + 1), (2 * width + 1,)]
    return [kinds[i % 5] for i in range(case['tensors'])]


def _row_sizes(shape, g):
    """Rows differ in size by orders of magnitude, as those of rare and of popular items do."""
    z = torch.randn((shape[0],) + (1,) * (len(shape) - 1), device=DEVICE, generator=g)
    return torch.exp(1.5 * z - 6.0)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device=DEVICE, generator=g)

    def codes(*shape):
        return torch.randint(-127, 128, shape, device=DEVICE, generator=g, dtype=torch.int8)

    state = {'case': case}
    if case['op'] == 'adamw':
        dtype = DTYPES[case['dtype']]
        for key in ('params', 'grads', 'm', 'v', 'steps', 'scales'):
            state[key] = []
        for shape in _shapes(case):
            size = _row_sizes(shape, g)
            m, v = 0.3 * size * normal(*shape), size * size * (0.2 + 0.3 * normal(*shape).square())
            state['params'].append((0.1 * normal(*shape)).to(dtype))
            state['grads'].append((size * normal(*shape)).to(dtype))
            state['steps'].append(torch.full((), float(STEP), device=DEVICE))
            if case['bits'] == 8:
                half = torch.full((1,), 0.5, device=DEVICE)
                m8, ms = _encode(m, half, 4, 448.0)
                v8, vs = _encode(v, half, 5, 57344.0)
                state['m'].append(m8.view(torch.float8_e4m3fn))
                state['v'].append(v8.view(torch.float8_e5m2))
                state['scales'].append(torch.stack([ms, vs], 1).contiguous())
            else:
                state['m'].append(m)
                state['v'].append(v)
        return state
    if case['op'] == 'quantize':
        shape = (case['rows'], case['width'])
        state['x'] = (_row_sizes(shape, g) * 40 * normal(*shape)).to(DTYPES[case['dtype']])
        return state
    m, n, k = case['m'], case['n'], case['k']
    state['b'], state['b_scale'] = codes(n, k), torch.exp(0.3 * normal(n) - 7.0)
    state['bias'] = 0.1 * normal(n) if case['bias'] else None
    if case['op'] == 'linear':
        state['x'] = normal(m, k).to(DTYPES[case['dtype']])
    else:
        state['a'], state['a_scale'] = codes(m, k), torch.exp(0.3 * normal(m) - 5.0)
    return state


# ---- the operators' plain forms ------------------------------------------------------------------------------------------------
_M32 = 0xFFFFFFFF


def _mix(x):
    """A 32-bit mixing function on int64 values."""
    x = x ^ (x >> 16)
    x = (x * 0x21f0aaad) & _M32
    x = x ^ (x >> 15)
    x = (x * 0x735a2d97) & _M32
    return x ^ (x >> 15)


def _uniforms(n, index, step):
    """Two numbers in (0, 1), of 16 bits each, for every element of tensor `index` at step `step` (a tensor of one value)."""
    key = _mix(_mix(step.to(torch.int64) ^ (SEED & _M32)) ^ ((SEED >> 32) + index * 0x9e3779b9 & _M32))
    i = torch.arange(n, device=DEVICE)
    h = _mix((i ^ _mix(key ^ (i >> 32))) & _M32)
    return ((h & 0xFFFF).float() + 0.5) / 65536.0, ((h >> 16).float() + 0.5) / 65536.0


def _encode(x, u, exponent_bits, top):
    """x in blocks of BLOCK elements as 8-bit floating codes of the block's largest magnitude (which becomes `top`), rounded up
    with the probability of the part cut off (where u says so); (codes uint8 like x, scales [blocks])."""
    mantissa, bias = 7 - exponent_bits, (1 << (exponent_bits - 1)) - 1
    flat = x.reshape(-1)
    n = flat.numel()
    rows = torch.nn.functional.pad(flat, (0, -n % BLOCK)).reshape(-1, BLOCK)
    big = rows.abs().amax(1)
    some = big >= 2.0 ** -100
    t = (rows.abs() * torch.where(some, top / big, 0.0)[:, None]).reshape(-1)[:n]
    e = torch.clamp((t.view(torch.int32) >> 23) - (127 - bias), min=1)
    k = torch.floor(torch.ldexp(t, mantissa + bias - e) + u).to(torch.int32)
    code = ((e - 1) << mantissa) + k
    if exponent_bits == 5:
        code = torch.maximum(code, (t > 0).to(torch.int32))          # a second moment that is not zero stays so
    code = code + 128 * ((flat < 0) & (code > 0)).to(torch.int32)
    return code.to(torch.uint8).reshape(x.shape), torch.where(some, big / top, 0.0)


def _decode(codes, scale):
    flat = codes.reshape(-1).float()
    return (flat * scale.repeat_interleave(BLOCK)[:flat.numel()]).reshape(codes.shape)


def _adamw_one(state, i, factor):
    """Tensor i of the list: moments and parameter are rewritten in place."""
    bits = state['case']['bits']
    p, step = state['params'][i], state['steps'][i]
    step += 1
    g = state['grads'][i].float() * factor
    m, v = state['m'][i], state['v'][i]
    m0, v0 = (m, v) if bits == 32 else (_decode(m, state['scales'][i][:, 0]), _decode(v, state['scales'][i][:, 1]))
    m1, v1 = BETA1 * m0 + (1 - BETA1) * g, BETA2 * v0 + (1 - BETA2) * g * g
    c1, c2 = 1 - BETA1 ** step.double(), 1 - BETA2 ** step.double()
    denom = torch.sqrt(v1) / torch.sqrt(c2).float() + EPS
    p.copy_(p.float() * (1 - LR * DECAY) - (LR / c1).float() * (m1 / denom))
    if bits == 32:
        m.copy_(m1)
        v.copy_(v1)
    else:
        um, uv = _uniforms(p.numel(), i, step)
        m8, ms = _encode(m1, um, 4, 448.0)
        v8, vs = _encode(v1, uv, 5, 57344.0)
        m.view(torch.uint8).copy_(m8)
        v.view(torch.uint8).copy_(v8)
        state['scales'][i].copy_(torch.stack([ms, vs], 1))


def _adamw(state):
    norm, factor = None, 1.0
    if state['case']['clip']:
        norm = torch.sqrt(sum(g.double().square().sum() for g in state['grads']))
        factor = torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0).float()
        norm = norm.float()
    for i in range(len(state['params'])):
        _adamw_one(state, i, factor)
    return norm


def _quantize(x):
    x = x.float()
    scale = (x.abs().amax(1).double() / 127).float()
    q = torch.round(x.double() / torch.where(scale > 0, scale, 1.0).double()[:, None])       # next to a border 64 bits decide
    return torch.clamp(q, -127, 127).to(torch.int8), scale


def _product(a, a_scale, b, b_scale, bias, dtype):
    exact = torch.float32 if a.shape[1] <= 1024 else torch.float64       # whole numbers: sums under 2^24 are exact in 32 bits
    y = (a.to(exact) @ b.to(exact).t()).float() * a_scale[:, None] * b_scale
    return (y if bias is None else y + bias).to(dtype)


# ---- one pass ------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state['case']
    if own:
        from igcn_cf_amd import ops
    if case['op'] == 'adamw':
        if own:
            norm = ops.adamw_step(state['params'], state['grads'], state['m'], state['v'], state['steps'], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                                  weight_decay=DECAY, max_grad_norm=MAX_NORM if case['clip'] else None,
                                  scales=state['scales'] if case['bits'] == 8 else None, seed=SEED)
        else:
            norm = _adamw(state)
        out = {'p': state['params'], 'm': state['m'], 'v': state['v'], 'scale': state['scales']}
        return out if norm is None else dict(out, norm=norm)
    if case['op'] == 'quantize':
        if own:
            q, scale = ops.quantize_rows_i8(state['x'])
            return {'values': ops.dequantize_rows_i8(q, scale), 'scale': scale}
        q, scale = _quantize(state['x'])
        return {'values': q.float() * scale[:, None], 'scale': scale}
    dtype = DTYPES[case['out']]
    if case['op'] == 'linear':
        if own:
            return ops.linear_i8(state['x'], state['b'], state['b_scale'], bias=state['bias'], dtype=dtype)
        return _product(*_quantize(state['x']), state['b'], state['b_scale'], state['bias'], dtype)
    if own:
        return ops.matmul_i8(state['a'], state['a_scale'], state['b'], state['b_scale'], bias=state['bias'], dtype=dtype)
    return _product(state['a'], state['a_scale'], state['b'], state['b_scale'], state['bias'], dtype)


def work(case):
    if case['op'] == 'adamw':
        n = sum(math.prod(s) for s in _shapes(case))
        size = 4 if case['dtype'] == 'float32' else 2
        moments = 16 if case['bits'] == 32 else 4 + 16 / BLOCK
        return {'bytes': n * (3 * size + moments), 'flops': 15 * n}
    if case['op'] == 'quantize':
        n = case['rows'] * case['width']
        return {'bytes': n * ((4 if case['dtype'] == 'float32' else 2) + 1 + 4) + 4 * case['rows'], 'flops': 3 * n}
    m, n, k = case['m'], case['n'], case['k']
    a = m * k * {'float32': 4, 'bfloat16': 2, 'float16': 2}[case['dtype']] if case['op'] == 'linear' else m * k + 4 * m
    out = 4 if case['out'] == 'float32' else 2
    return {'bytes': a + n * k + m * n * out + 4 * n * (2 if case['bias'] else 1), 'flops': 2 * m * n * k}


# ---- what the definitions say, in 64 bits --------------------------------------------------------------------------------------
def _hash64(v):
    """The mixing function, on int64 tensors, its products taken in 16-bit halves."""
    def times(x, c):
        return ((x & 0xFFFF) * c + ((((x >> 16) * c) & 0xFFFF) << 16)) % (1 << 32)
    v = v ^ torch.div(v, 1 << 16, rounding_mode='floor')
    v = times(v, 0x21f0aaad)
    v = v ^ torch.div(v, 1 << 15, rounding_mode='floor')
    v = times(v, 0x735a2d97)
    return v ^ torch.div(v, 1 << 15, rounding_mode='floor')


def _exact_moment(x, u, top, smallest, digits, keep):
    """Rounds x / (block's maximum / top) to `digits` binary digits behind the first (multiples of `smallest` at least), up where the
    part cut off and u make one; float64 values and scales."""
    n = x.numel()
    whole = torch.zeros((n + BLOCK - 1) // BLOCK * BLOCK, dtype=torch.float64, device=DEVICE)
    whole[:n] = x.reshape(-1)
    big = whole.abs().reshape(-1, BLOCK).max(1).values
    scale = big / top
    ratio = (whole.abs() / torch.where(scale > 0, scale, 1.0).repeat_interleave(BLOCK))[:n]
    quantum = torch.pow(2.0, torch.floor(torch.log2(torch.clamp(ratio, min=1e-300))) - digits).clamp(min=smallest)
    up = torch.floor(ratio / quantum + u) * quantum
    if keep:
        up = torch.where((up == 0) & (ratio > 0), smallest, up)
    return (up * torch.sign(x.reshape(-1))).reshape(x.shape), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'adamw':
        factor, out = 1.0, {'p': [], 'm': [], 'v': [], 'scale': []}
        if case['clip']:
            norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s['grads']))
            factor = min(1.0, MAX_NORM / (norm + 1e-6))
            out['norm'] = norm
        t = STEP + 1
        for i, (p, g) in enumerate(zip(s['params'], s['grads'])):
            n = p.numel()
            m, v = s['m'][i].double(), s['v'][i].double()
            if case['bits'] == 8:
                block = torch.div(torch.arange(n, device=DEVICE), BLOCK, rounding_mode='floor')
                m = m * s['scales'][i][:, 0].double()[block].reshape(p.shape)
                v = v * s['scales'][i][:, 1].double()[block].reshape(p.shape)
            g = g.double() * factor
            m = m + (1 - BETA1) * (g - m)
            v = v + (1 - BETA2) * (g ** 2 - v)
            change = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
            out['p'].append(p.double() - LR * DECAY * p.double() - LR * change)
            if case['bits'] == 8:
                one = torch.zeros(1, dtype=torch.int64, device=DEVICE)
                key = _hash64(_hash64(one + (t ^ SEED)) ^ (index_key(i)))
                h = _hash64(torch.arange(n, device=DEVICE) ^ _hash64(key))
                m, ms = _exact_moment(m, ((h % 65536).double() + 0.5).div(65536), 448.0, 2.0 ** -9, 3, False)
                v, vs = _exact_moment(v, (torch.div(h, 65536, rounding_mode='floor').double() + 0.5).div(65536), 57344.0, 2.0 ** -16, 2, True)
                out['scale'].append(torch.stack([ms, vs], 1))
            out['m'].append(m)
            out['v'].append(v)
        return out
    if case['op'] == 'quantize':
        scale, values = _exact_rows(s['x'])
        return {'values': values, 'scale': scale}
    if case['op'] == 'linear':
        a_scale, a = _exact_rows(s['x'])
    else:
        a_scale, a = None, s['a'].double() * s['a_scale'].double().unsqueeze(1)
    y = torch.zeros(case['m'], case['n'], dtype=torch.float64, device=DEVICE)
    for k in range(0, case['k'], 512):
        y += torch.mm(a[:, k:k + 512], (s['b'][:, k:k + 512].double() * s['b_scale'].double().unsqueeze(1)).t().contiguous())
    return y if s['bias'] is None else y + s['bias'].double()


def index_key(i):
    return (0x9e3779b9 * i) % (1 << 32)


def _exact_rows(x):
    """(scales, the values the rows' codes stand for): the largest magnitude over 127, held in 32 bits, and its nearest multiples."""
    x = x.double()
    scale = (torch.linalg.vector_norm(x, ord=float('inf'), dim=1) / 127).float().double()
    q = x / torch.where(scale > 0, scale, 1.0).unsqueeze(1)
    down = torch.floor(q)
    odd, rest = torch.remainder(down, 2) == 1, q - down
    q = (down + ((rest > 0.5) | ((rest == 0.5) & odd)).double()).clamp(-127, 127)
    return scale, q * scale.unsqueeze(1)
