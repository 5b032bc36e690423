"""Attention over the 8-bit cache on the GPU, against plain implementations in 64 bits.

Tolerances count roundings: u(t) = finfo(t).eps / 2 is half a step of a type, relative to the value.
"""
import math

import pytest
import torch

from ishizuki_amd import attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LIMIT = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def u(dtype):
    return torch.finfo(dtype).eps / 2


def normal(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def make_batch(lengths, rows, blocks=None, width=None, seed=0, spare=2):
    """(batch on the GPU, blocks in the pool): sequences of the given tokens and new rows, blocks in a random order."""
    need = [-(-n // 64) for n in lengths]
    blocks = sum(need) + spare if blocks is None else blocks
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(max(need), 1) if width is None else width
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    starts = i32(0, *torch.tensor(rows).cumsum(0).tolist())
    return attention.Batch(table.to(DEV), i32(*lengths).to(DEV), starts.to(DEV), max(rows), max(lengths)), blocks


def random_cache(blocks, heads, dim, dtype, seed=0):
    """A pool of finite codes and scales of about a unit value."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((2, blocks, heads, 64 * dim), generator=g)
    scale = x.abs().amax(-1) / LIMIT[dtype]
    x = x / scale[..., None]
    codes = (x.round() if dtype is INT8 else x).to(dtype).view(INT8)
    c = attention.new_cache(blocks, heads, dim, dtype, device="cpu")
    c.k.view(INT8).copy_(codes[0].view(c.k.shape))
    c.v.view(INT8).copy_(codes[1].view(c.v.shape))
    return attention.Cache(c.k, c.v, scale[0].contiguous(), scale[1].contiguous())


def gpu(cache):
    return attention.Cache(*(t.to(DEV) for t in cache))


def values(cache, batch, s, length=None):
    """(k, v) [tokens, heads, dim] of sequence s in 64 bits, NaN where the table has no block."""
    length = int(batch.lengths[s]) if length is None else length
    blocks, heads, _, dim = cache.k.shape
    k = torch.full((length, heads, dim), float("nan"), dtype=torch.float64)
    v = k.clone()
    for j in range(-(-length // 64)):
        b = int(batch.table[s, j]) if j < batch.table.shape[1] else -1
        if not 0 <= b < blocks:
            continue
        n = min(64, length - 64 * j)
        k[64 * j:64 * j + n] = (cache.k[b].cpu().double() * cache.k_scale[b].cpu().double()[:, None, None])[:, :n].transpose(0, 1)
        v[64 * j:64 * j + n] = (cache.v[b].cpu().double() * cache.v_scale[b].cpu().double()[:, None, None])[:, :, :n].permute(2, 0, 1)
    return k, v


# ---------------------------------------------------------------- norms and rotation
def rope_reference(x, positions, inv_freq, weight, eps, interleaved, factor=1.0):
    """[rows, heads, dim] in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    rot = 2 * len(inv_freq)
    if rot == 0:
        return x
    angle = positions.double()[:, None, None] * torch.tensor(inv_freq, dtype=torch.float64)
    c, s = angle.cos() * factor, angle.sin() * factor
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = x.clone()
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


def rope_tolerance(y, x, weight, eps, dtype, factor=1.0):
    """Half a step of the output, and in fp32: the norm's sum of squares, root, quotient and two products (8 half steps;
    the sum's tree adds at most 8 more), the angle's cosine and sine (half a step of the phase's 2^-25 turns, 2 pi 2^-26,
    and 3 half steps of the series: 2^-23 in all), two products and a sum (3): below 2^-19 of the pair's size."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    size = x.abs().amax(-1, keepdim=True) * math.sqrt(2) * factor
    return u(dtype) * y.abs() + 2.0 ** -19 * size + (2.0 ** -25 if dtype is F16 else 1e-38)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,rot,interleaved", [(64, 64, False), (128, 128, False), (256, 64, True), (128, 32, False),
                                                 (256, 256, False), (64, 16, True), (128, 0, False)])
@pytest.mark.parametrize("rows,heads,kv", [(1, 5, 1), (7, 32, 8), (2049, 3, 2)])
def test_norm_rope(dtype, dim, rot, interleaved, rows, heads, kv):
    print(f"norm_rope {dtype} {rows} x ({heads}, {kv}) x {dim} rot {rot}", flush=True)
    qkv = normal(1, rows, heads + 2 * kv, dim, dtype=dtype)
    positions = torch.arange(rows, dtype=torch.int32) * 977 + 1000003
    inv = [1e6 ** (-2.0 * i / max(rot, 1)) for i in range(rot // 2)]
    wq, wk = 1 + normal(2, dim) / 4, 1 + normal(3, dim) / 4
    d = qkv.to(DEV)
    table = attention.turns(inv_freq=inv, device=DEV) if rot else None
    q, k = attention.norm_rope(d[:, :heads], d[:, heads:heads + kv], positions.to(DEV), table, wq.to(DEV), wk.to(DEV),
                               eps=1e-5, interleaved=interleaved, factor=1.25)
    for got, x, w in ((q, qkv[:, :heads], wq), (k, qkv[:, heads:heads + kv], wk)):
        y = rope_reference(x, positions, inv, w, 1e-5, interleaved, 1.25)
        assert torch.all((got.cpu().double() - y).abs() <= rope_tolerance(y, x, w, 1e-5, dtype, 1.25))


def test_norm_rope_parts():
    """No weight: no norm; no turns: no rotation; negative and far positions; a row of zeros; in place through the C call's
    own rules; k heads alone."""
    x = normal(4, 5, 2, 128, dtype=F16)
    x[3] = 0
    d, positions = x.to(DEV), i32(-3, 0, 5, 7, 2 ** 31 - 1)
    inv = [1e4 ** (-2.0 * i / 128) for i in range(64)]
    q, k = attention.norm_rope(d, d)
    assert torch.equal(q, d) and torch.equal(k, d)
    q, k = attention.norm_rope(d, d[:, :1], positions.to(DEV), attention.turns(inv_freq=inv, device=DEV))
    y = rope_reference(x, positions, inv, None, 0, False)
    assert torch.all((q.cpu().double() - y).abs() <= rope_tolerance(y, x, None, 0, F16) + 2.0 ** -20 * x.double().abs().amax())
    assert torch.equal(k, q[:, :1]) and torch.all(q[3] == 0)
    w = torch.full((128,), 2.0, device=DEV)
    q, k = attention.norm_rope(d[:, :0], d, k_weight=w)
    y = rope_reference(x, positions, [], w.cpu(), 1e-6, False)
    assert q.shape == (5, 0, 128)
    assert torch.all((k.cpu().double() - y).abs() <= rope_tolerance(y, x, w.cpu(), 1e-6, F16))


# ---------------------------------------------------------------- writing and reading
class Model:
    """The cache in 64 bits on the CPU: codes [blocks, heads, 64, dim] as numbers, scales; appends as the header says."""

    def __init__(self, cache):
        self.dtype = cache.k.dtype
        self.held = [cache.k.cpu().double(), cache.v.cpu().double().transpose(-1, -2).contiguous()]
        self.scale = [cache.k_scale.cpu().double(), cache.v_scale.cpu().double()]
        self.ratio = [torch.full_like(x, math.nan) for x in self.held]  # of what was coded since the last check

    def code(self, x):
        m = LIMIT[self.dtype]
        x = x.clamp(-m, m)
        if self.dtype is INT8:
            return x.round()
        step = 2.0 ** (torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        return (x / step).round() * step

    def append(self, which, new, table, first):
        """new [rows, heads, dim] at positions first.. of the sequence whose blocks `table` lists."""
        for j in sorted({(first + i) // 64 for i in range(new.shape[0]) if first + i >= 0}):
            b = table[j] if j < len(table) else -1
            if not 0 <= b < self.held[0].shape[0]:
                continue
            rows = [i for i in range(new.shape[0]) if (first + i) // 64 == j and first + i >= 0]
            slots = [(first + i) % 64 for i in rows]
            x = new[rows].double()
            for h in range(x.shape[1]):
                amax = float(x[:, h].abs().max()) if torch.isfinite(x[:, h]).all() else math.nan
                s = float(self.scale[which][b, h])
                if math.isnan(amax):
                    s = math.nan
                elif slots[0] == 0:
                    s = max(amax / LIMIT[self.dtype], 2.0 ** -126)
                else:
                    s = max(s, 2.0 ** -126) if s == s else s
                    k = 0
                    while amax > LIMIT[self.dtype] * s * 2.0 ** k * (1 + 2.0 ** -22):
                        k += 1
                    s *= 2.0 ** k
                    if k:
                        self.held[which][b, h, :slots[0]] = self.code(self.held[which][b, h, :slots[0]] / 2.0 ** k)
                self.scale[which][b, h] = s
                self.ratio[which][b, h, slots] = x[:, h] / s
                self.held[which][b, h, slots] = 0.0 if math.isnan(s) else self.code(x[:, h] / s)

    def check(self, cache, key_error=0.0):
        """Scales to two half steps of fp32 (a quotient), codes equal but where x / s lies within fp32's roundings of the
        border between two neighbours (a quotient or a reciprocal and a product: four half steps); keys that were computed
        may be off by `key_error` of their head's largest before they are coded. Then goes on from what the GPU holds."""
        got = [cache.k.cpu().double(), cache.v.cpu().double().transpose(-1, -2).contiguous()]
        for which, scale in enumerate((cache.k_scale, cache.v_scale)):
            a, b = scale.cpu().double(), self.scale[which]
            off = 0.0 if which else key_error
            assert torch.equal(a.isnan(), b.isnan())
            assert torch.all(((a - b).abs() <= (2 * u(F32) + off) * b)[~b.isnan()])
            x, y, ratio = got[which], self.held[which], self.ratio[which]
            differ = x != y
            near = (ratio - (x + y) / 2).abs() <= 4 * u(F32) * ratio.abs() + 2 * off * LIMIT[self.dtype]
            assert torch.all(near[differ]), float(differ.double().mean())
            step = 1.0 if self.dtype is INT8 else 2.0 ** (torch.floor(torch.log2(torch.minimum(x.abs(), y.abs()).clamp(min=2.0 ** -6))) - 3)
            assert torch.all((x - y).abs() <= step)
            self.held[which], self.scale[which] = x, a
            self.ratio[which] = torch.full_like(x, math.nan)


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("x", [F16, BF16, F32])
@pytest.mark.parametrize("heads,dim", [(3, 64), (8, 128), (1, 256)])
def test_append_and_read(dtype, x, heads, dim):
    """Ragged sequences written in several calls: fresh and partly filled blocks, one token and many, scales that grow."""
    print(f"append {dtype} {x} {heads} x {dim}", flush=True)
    calls = [[63, 0, 130, 1], [1, 0, 1, 70], [1, 5, 64, 1], [200, 1, 1, 0]]
    total = [sum(c[s] for c in calls) for s in range(4)]
    whole, blocks = make_batch(total, [0] * 4, seed=dim)
    cache = random_cache(blocks, heads, dim, dtype, seed=7)
    model, cache = Model(cache), gpu(cache)
    held = [0] * 4
    for n, rows in enumerate(calls):
        size = 3.0 ** n  # later tokens are larger
        k, v = (normal(10 * n + i, sum(rows), heads, dim) * size for i in (1, 2))
        k[:, :, ::17] *= 6
        k, v = k.to(x), v.to(x)
        starts = [0, *torch.tensor(rows).cumsum(0).tolist()]
        held = [h + r for h, r in zip(held, rows)]
        batch = whole._replace(lengths=i32(*held).to(DEV), starts=i32(*starts).to(DEV), max_rows=max(rows))
        assert attention.append(k.to(DEV), v.to(DEV), cache, batch) is True
        for s in range(4):
            for which, t in enumerate((k, v)):
                model.append(which, t[starts[s]:starts[s + 1]], whole.table[s].tolist(), held[s] - rows[s])
        model.check(cache)
    for out in (F16, BF16, F32):
        for tail in (1, 63, 64, 65, max(held) + 9):
            got = attention.read(cache, batch, tail=tail, dtype=out)
            for s in range(4):
                for y, ref in zip(got, values(cache, batch, s)):
                    y, ref = y[s].cpu(), ref[-tail:]
                    assert torch.all(y[:tail - ref.shape[0]] == 0)
                    y = y[tail - ref.shape[0]:].double()
                    # a product of 24 and 8 bits rounded to fp32 and then to the output
                    assert torch.all((y - ref).abs() <= (u(out) + u(F32)) * ref.abs() + (2.0 ** -25 if out is F16 else 0))


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("dim,rot,interleaved", [(128, 128, False), (64, 32, True), (256, 64, False)])
def test_append_with_norms_and_rotation(dtype, dim, rot, interleaved):
    rows, lengths, heads, kv = [1, 90, 0, 3], [40, 90, 0, 130], 6, 2
    batch, blocks = make_batch(lengths, rows, seed=3)
    cache = random_cache(blocks, kv, dim, dtype, seed=8)
    model, cache = Model(cache), gpu(cache)
    qkv = normal(5, sum(rows), heads + 2 * kv, dim, dtype=BF16)
    positions = torch.cat([torch.arange(n - r, n) for n, r in zip(lengths, rows)]).int() + 500000
    inv = [1e4 ** (-2.0 * i / rot) for i in range(rot // 2)]
    wq, wk = 1 + normal(2, dim) / 4, 2 + normal(3, dim) / 4
    d = qkv.to(DEV)
    q = attention.append(d[:, heads:heads + kv], d[:, heads + kv:], cache, batch, q=d[:, :heads],
                         positions=positions.to(DEV), turns=attention.turns(inv_freq=inv, device=DEV), q_weight=wq.to(DEV),
                         k_weight=wk.to(DEV), interleaved=interleaved)
    y = rope_reference(qkv[:, :heads], positions, inv, wq, 1e-6, interleaved)
    assert torch.all((q.cpu().double() - y).abs() <= rope_tolerance(y, qkv[:, :heads], wq, 1e-6, BF16))
    k = rope_reference(qkv[:, heads:heads + kv], positions, inv, wk, 1e-6, interleaved)
    at = 0
    for s, r in enumerate(rows):
        for which, t in enumerate((k, qkv[:, heads + kv:])):
            model.append(which, t[at:at + r], batch.table[s].tolist(), lengths[s] - r)
        at += r
    model.check(cache, key_error=2.0 ** -18)  # see rope_tolerance: 2^-19 sqrt 2 of the head's largest


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 9, 31])
def test_append_takes_scales_from_normed_keys(dtype, dim, rows):
    """Keys far larger before their norm than after it, into partly filled blocks whose scales hold the latter: the scales
    stay. The same keys without a norm make them grow."""
    batch, blocks = make_batch([20 + rows, 61 + rows], [rows, rows], seed=3)
    first = random_cache(blocks, 2, dim, dtype, seed=8)
    k = normal(5, 2 * rows, 2, dim, dtype=BF16) * 50
    w = torch.full((dim,), 0.5)
    for weight in (w, None):
        cache = gpu(first)
        model = Model(cache)
        x = rope_reference(k, None, [], weight, 1e-6, False)
        attention.append(k.to(DEV), k.to(DEV), cache, batch, k_weight=None if weight is None else weight.to(DEV))
        for s in range(2):
            for which, new in enumerate((x, k)):
                model.append(which, new[s * rows:s * rows + rows], batch.table[s].tolist(), (20, 61)[s])
        model.check(cache, key_error=2.0 ** -18)
        grown = cache.k_scale[batch.table[0, 0].item()].cpu() > first.k_scale[batch.table[0, 0].item()]
        assert bool(grown.any()) == (weight is None)


def test_append_again_changes_nothing():
    batch, blocks = make_batch([70, 3], [7, 2])
    cache = gpu(random_cache(blocks, 2, 128, INT8, seed=9))
    k, v = normal(1, 9, 2, 128).to(DEV) * 20, normal(2, 9, 2, 128).to(DEV)
    attention.append(k, v, cache, batch)
    once = [t.clone() for t in cache]
    attention.append(k, v, cache, batch)
    assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(once, cache))


@pytest.mark.parametrize("dtype", [INT8, E4M3])
def test_append_of_what_is_not_a_number(dtype):
    """An infinity or NaN shows as NaN in its block and head alone; zeros and the smallest values are codes of 0."""
    batch, blocks = make_batch([128, 64], [128, 64])
    cache = gpu(random_cache(blocks, 3, 64, dtype))
    k, v = normal(1, 192, 3, 64), normal(2, 192, 3, 64)
    k[5, 1, 7], v[70, 2, 0] = math.inf, math.nan
    k[128:, 0] = 0
    v[128:, 1] = 1e-45
    attention.append(k.to(DEV), v.to(DEV), cache, batch)
    gk, gv = attention.read(cache, batch, dtype=F32)
    bad_k, bad_v = torch.zeros(2, 128, 3, 64, dtype=torch.bool), torch.zeros(2, 128, 3, 64, dtype=torch.bool)
    bad_k[0, :64, 1], bad_v[0, 64:, 2] = True, True
    assert torch.equal(gk.cpu().isnan(), bad_k) and torch.equal(gv.cpu().isnan(), bad_v)
    assert torch.all(gk[1, :, 0] == 0) and torch.all(gv[1, :, 1] == 0)
    attention.append(k[128:].to(DEV), v[128:].to(DEV), cache, batch._replace(starts=i32(0, 64, 64).to(DEV), lengths=i32(64, 0).to(DEV)))
    assert torch.isfinite(cache.k_scale[batch.table[0, 0].item()]).all()  # started again


def test_append_leaves_the_rest_alone():
    """Holes of the table, tokens past it, rows past max_rows' blocks and other blocks stay as they were."""
    table = i32(2, -1, 99, 5).view(1, 4).to(DEV)
    batch = attention.Batch(table, i32(300).to(DEV), i32(0, 290).to(DEV), 290, 300)
    cache = gpu(random_cache(8, 2, 64, INT8))
    before = attention.Cache(*(t.clone() for t in cache))
    model = Model(cache)
    k, v = normal(1, 290, 2, 64), normal(2, 290, 2, 64)
    attention.append(k.to(DEV), v.to(DEV), cache, batch)
    # 300 tokens are cut at the table's 256: the rows are then the last 290 of those, the first 34 of them nowhere
    for which, t in enumerate((k, v)):
        model.append(which, t, [2, -1, 99, 5], 256 - 290)
    model.check(cache)
    for b in (0, 1, 3, 4, 6, 7):
        assert torch.equal(cache.k[b], before.k[b]) and torch.equal(cache.v[b], before.v[b])


# ---------------------------------------------------------------- attention
def attention_reference(q, cache, batch, scale, causal, window):
    """(out, bound) [rows, heads, dim] in 64 bits: bound is sum of weights |v|, and what the logits' roundings move."""
    blocks, heads, _, dim = cache.k.shape
    group = q.shape[1] // heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound, shift = torch.zeros_like(out), torch.zeros(q.shape[0], q.shape[1], 1, dtype=torch.float64)
    starts = batch.starts.tolist()
    for s in range(len(starts) - 1):
        n, length = starts[s + 1] - starts[s], min(int(batch.lengths[s]), 64 * batch.table.shape[1])
        k, v = values(cache, batch, s, length)
        hole = torch.tensor([not 0 <= int(batch.table[s, t // 64]) < blocks for t in range(length)], dtype=torch.bool)
        k[hole], v[hole] = 0, 0
        token = torch.arange(length)
        for i in range(n):
            at = length - n + i
            seen = ~hole
            if causal:
                seen = seen & (token <= at)
                if window:
                    seen = seen & (token > at - window)
            if not seen.any():
                continue
            for h in range(heads):
                x = q[starts[s] + i, h * group:(h + 1) * group].double()
                logit = x @ k[seen, h].T * scale
                w = torch.softmax(logit, -1)
                out[starts[s] + i, h * group:(h + 1) * group] = w @ v[seen, h]
                bound[starts[s] + i, h * group:(h + 1) * group] = w @ v[seen, h].abs()
                shift[starts[s] + i, h * group:(h + 1) * group, 0] = (x.abs() @ k[seen, h].abs().T * scale).amax(-1)
    return out, bound, shift


def attention_close(got, q, ref):
    """Half a step of the output's type; of each weight half a step of fp16 (2^-11), exp2 and the sums in fp32 (2^-20 in
    all), weights below fp16's normals 2^-25 of the largest each; a logit's sum of dim products and three scalings, and q's
    fp16 image (2^-25 of a row's largest a value): dim + 8 half steps of the products' sizes, twice (numerator and sum)."""
    out, bound, shift = ref
    dim = q.shape[-1]
    tol = u(got.dtype) * out.abs() + (2.0 ** -11 + 2.0 ** -20 + 2 * (dim + 8) * u(F32) * shift) * bound
    tol = tol + 2.0 ** -25 * bound.amax() * 64 + (2.0 ** -25 if got.dtype is F16 else 0)
    d = (got.cpu().double() - out).abs()
    assert torch.all(d <= tol), float((d / tol).max())


CASES = [  # lengths, rows, causal, window
    ([1], [1], True, 0), ([64], [1], True, 0), ([65], [1], True, 0), ([777], [1], True, 0), ([5000], [1], True, 0),
    ([0, 130, 63, 64], [0, 1, 1, 1], True, 0), ([200, 77], [5, 3], True, 0), ([129, 64], [129, 64], True, 0),
    ([300], [41], True, 100), ([1000, 70, 9], [2, 70, 1], True, 33), ([513], [3], True, 1), ([200, 1, 0], [7, 33, 0], False, 0),
    ([20], [37], True, 0), ([150], [150], True, 64),
]


@pytest.mark.parametrize("lengths,rows,causal,window", CASES)
@pytest.mark.parametrize("heads,group,dim,dtype,x", [(2, 4, 128, INT8, BF16), (1, 1, 64, E4M3, F16), (3, 5, 64, INT8, F16),
                                                     (2, 8, 256, E4M3, BF16), (1, 16, 128, E4M3, F16), (1, 3, 256, INT8, BF16)])
def test_attend(lengths, rows, causal, window, heads, group, dim, dtype, x):
    print(f"attend {lengths} {rows} {causal} {window} {heads} x {group} x {dim} {dtype} {x}", flush=True)
    batch, blocks = make_batch(lengths, rows, seed=1)
    cache = random_cache(blocks, heads, dim, dtype, seed=sum(lengths))
    q = normal(3, sum(rows), heads * group, dim, dtype=x)
    got = attention.attend(q.to(DEV), gpu(cache), batch, causal=causal, window=window)
    attention_close(got, q, attention_reference(q, cache, batch, dim ** -0.5, causal, window))
    again = attention.attend(q.to(DEV), gpu(cache), batch, causal=causal, window=window)
    assert torch.equal(got, again)


def test_attend_sharp_and_large():
    """Logits of some hundreds: one token takes all the weight, nothing overflows; queries beyond fp16's range."""
    batch, blocks = make_batch([500], [3], seed=1)
    cache = random_cache(blocks, 2, 128, INT8, seed=5)
    q = normal(3, 3, 4, 128) * 3e5
    q = q.to(BF16)
    got = attention.attend(q.to(DEV), gpu(cache), batch, scale=1e-3)
    attention_close(got, q, attention_reference(q, cache, batch, 1e-3, True, 0))


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("dtype", [INT8, E4M3])
def test_attend_ignores_what_it_does_not_see(dtype, rows):
    """NaN scales of blocks that no row of a tile sees, or that one row does not; NaN codes and whatever else past the
    end; holes in the table."""
    batch, blocks = make_batch([300], [rows], seed=2, width=9)
    cache = random_cache(blocks, 2, 64, dtype, seed=6)
    q = normal(3, rows, 4, 64, dtype=F16)
    batch.table[0, 1], batch.table[0, 2] = -1, blocks + 5
    ref = attention_reference(q, cache, batch, 0.125, True, 0)
    last = int(batch.table[0, 4])
    cache.k.view(INT8)[last, :, 300 - 256:] = 0x7F  # e4m3's NaN
    cache.v.view(INT8)[last, :, :, 300 - 256:] = 0x7F
    for b in range(blocks):
        if b not in batch.table[0].tolist():
            cache.k_scale[b], cache.v_scale[b] = math.nan, math.inf
    got = attention.attend(q.to(DEV), gpu(cache), batch)
    attention_close(got, q, ref)
    # the last block's scales of no number reach the rows that see it, and no others
    cache.k_scale[last], cache.v_scale[last] = math.nan, math.nan
    got = attention.attend(q.to(DEV), gpu(cache), batch).cpu()
    sees = torch.arange(300 - rows, 300) >= 256
    assert torch.equal(got.isnan(), sees[:, None, None].expand_as(got))
    if (~sees).any():
        keep = tuple(t[~sees] for t in ref)
        attention_close(got[~sees], q, keep)
    got = attention.attend(q.to(DEV), gpu(cache), batch, window=5).cpu()
    first = torch.arange(300 - rows, 300) < 256  # those rows' window lies before the last block
    assert not got[first].isnan().any()


WIDE = [  # lengths, rows, causal, window: what the kernels for more rows, longer caches and several splits get to see
    ([700], [33], True, 0), ([4500, 300], [20, 17], True, 0), ([9000], [70], True, 0), ([8300, 9000], [40, 66], True, 500),
    ([1030], [1030], True, 0), ([1500], [130], False, 0), ([5000], [9], True, 0), ([400, 1000], [1, 1], True, 0),
]


@pytest.mark.parametrize("lengths,rows,causal,window", WIDE)
@pytest.mark.parametrize("heads,group,dim,dtype,x", [(1, 4, 128, INT8, BF16), (2, 1, 64, E4M3, F16), (1, 2, 256, INT8, F16),
                                                     (1, 7, 64, INT8, BF16)])
def test_attend_longer(lengths, rows, causal, window, heads, group, dim, dtype, x):
    print(f"attend {lengths} {rows} {causal} {window} {heads} x {group} x {dim} {dtype} {x}", flush=True)
    batch, blocks = make_batch(lengths, rows, seed=1)
    cache = random_cache(blocks, heads, dim, dtype, seed=sum(lengths))
    q = normal(3, sum(rows), heads * group, dim, dtype=x)
    got = attention.attend(q.to(DEV), gpu(cache), batch, causal=causal, window=window)
    attention_close(got, q, attention_reference(q, cache, batch, dim ** -0.5, causal, window))


@pytest.mark.parametrize("lengths,rows,window", [([9000, 70], [1, 1], 1000), ([5000], [1], 64), ([20000], [1], 257),
                                                 ([12000, 3], [8, 3], 700), ([6000, 9000], [40, 8], 1500)])
@pytest.mark.parametrize("heads,group,dim,dtype,x", [(2, 4, 128, INT8, BF16), (2, 3, 64, E4M3, F16), (2, 2, 256, E4M3, BF16)])
def test_attend_window_of_a_long_cache(lengths, rows, window, heads, group, dim, dtype, x):
    print(f"attend {lengths} {rows} {window} {heads} x {group} x {dim} {dtype} {x}", flush=True)
    batch, blocks = make_batch(lengths, rows, seed=1)
    cache = random_cache(blocks, heads, dim, dtype, seed=sum(lengths))
    q = normal(3, sum(rows), heads * group, dim, dtype=x)
    got = attention.attend(q.to(DEV), gpu(cache), batch, window=window)
    attention_close(got, q, attention_reference(q, cache, batch, dim ** -0.5, True, window))


def test_attend_many_blocks_a_workgroup():
    """Caches of more blocks than a wave holds the numbers of, not split, with holes."""
    n, length = 64, 4500
    batch, blocks = make_batch([length] * n, [18] * n, seed=1)
    batch.table[:, 3], batch.table[5, 61:64], batch.table[:, 65] = -1, blocks, -7
    cache = random_cache(blocks, 4, 64, INT8, seed=7)
    q = normal(3, 18 * n, 4, 64, dtype=F16)
    got = attention.attend(q.to(DEV), gpu(cache), batch)
    for s in (0, 5, 63):
        one = attention.Batch(batch.table[s:s + 1], i32(length), i32(0, 18), 18, length)
        rows = slice(18 * s, 18 * s + 18)
        attention_close(got[rows], q[rows], attention_reference(q[rows], cache, one, 0.125, True, 0))


def visible(cache, batch, rows, length, window, group):
    """Sums of |v| over the tokens that each row sees, [rows, q heads, dim] in 64 bits."""
    _, v = values(cache, batch, 0, length)
    total = torch.cat((torch.zeros_like(v[:1]), v.abs().nan_to_num().cumsum(0)))
    end = length - rows + torch.arange(rows) + 1
    begin = (end - window).clamp(min=0) if window else torch.zeros_like(end)
    return (total[end] - total[begin]).repeat_interleave(group, 1)


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("rows,window", [(3, 0), (300, 0), (300, 20), (640, 64), (40, 7)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attend_value_scales_far_apart(dtype, rows, window, dim):
    """Blocks whose values differ by up to 2^100, and one that is all zeros with scales of 0: a row that sees none of the
    large ones is as exact as if they were not there. Weights below fp16's normals are off by 2^-25 of the largest each."""
    length = 640
    batch, blocks = make_batch([length], [rows], seed=2)
    cache = random_cache(blocks, 1, dim, dtype, seed=6)
    for j, e in enumerate([0, -30, 12, -45, 3, -3, 40, -60, 0, 9]):
        cache.v_scale[batch.table[0, j].item()] *= 2.0 ** e
    zero = batch.table[0, 4].item()
    cache.v_scale[zero], cache.k_scale[zero] = 0, 0
    cache.v.view(INT8)[zero] = 0
    q = normal(3, rows, 2, dim, dtype=BF16)
    out, bound, shift = attention_reference(q, cache, batch, dim ** -0.5, True, window)
    got = attention.attend(q.to(DEV), gpu(cache), batch, window=window).cpu().double()
    tol = u(BF16) * out.abs() + (2.0 ** -11 + 2.0 ** -19 + 2 * (dim + 8) * u(F32) * shift) * bound
    tol = tol + 2.0 ** -25 * visible(cache, batch, rows, length, window, 2) + 2.0 ** -126
    d = (got - out).abs()
    assert torch.all(d <= tol), float((d / tol).max())


def test_strides_streams_and_rows_of_no_sequence():
    batch, blocks = make_batch([100, 40], [2, 3], seed=4)
    cache = random_cache(blocks, 2, 128, INT8, seed=6)
    wide = normal(3, 9, 11, 128, dtype=F16)
    q = wide[::1, 1:7]
    ref = attention_reference(q[:5], cache, batch, 128 ** -0.5, True, 0)
    c, d = gpu(cache), wide.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attention.attend(d[:, 1:7], c, batch)
    torch.cuda.current_stream().wait_stream(side)
    attention_close(got[:5], q, ref)
    half = torch.empty(5, 6, 2, 128, dtype=F16, device=DEV)
    half[:, :, 0] = d[:5, 1:7]
    attention_close(attention.attend(half[:, :, 0], c, batch), q, ref)


def test_offsets_past_32_bits():
    """Blocks whose codes lie more than 4 GiB into the pool, written, read and attended to."""
    heads, dim = 8, 256
    blocks = (1 << 32) // (heads * 64 * dim) + 6
    cache = attention.new_cache(blocks, heads, dim, E4M3, device=DEV)
    table = torch.arange(blocks - 1, blocks - 5, -1, dtype=torch.int32).view(1, 4).to(DEV)
    k, v = normal(1, 200, heads, dim, dtype=F16), normal(2, 200, heads, dim, dtype=F16)
    batch = attention.Batch(table, i32(200).to(DEV), i32(0, 200).to(DEV), 200, 200)
    attention.append(k.to(DEV), v.to(DEV), cache, batch)
    small = attention.Cache(*(t[-6:].cpu() for t in cache))
    near = batch._replace(table=table - (blocks - 6))
    for got, ref in zip(attention.read(cache, batch, dtype=F32), values(small, near, 0)):
        assert torch.all((got[0].cpu().double() - ref).abs() <= u(F32) * ref.abs())
    q = normal(3, 1, 8, dim, dtype=F16)
    one = batch._replace(starts=i32(0, 1).to(DEV), max_rows=1)
    got = attention.attend(q.to(DEV), cache, one)
    attention_close(got, q, attention_reference(q, small, near._replace(starts=i32(0, 1)), dim ** -0.5, True, 0))


def test_captured_step_follows_the_lengths():
    """A step (norms, rotation, writing, attention) captured once and replayed as the sequences grow gives what eager
    calls give, bit for bit."""
    heads, kv, dim = 8, 2, 128
    lengths, steps = [60, 127, 1], 6
    whole, blocks = make_batch([n + steps + 1 for n in lengths], [1, 1, 1], seed=5)
    first = gpu(random_cache(blocks, kv, dim, INT8, seed=2))
    table = attention.turns(dim, device=DEV)
    w = torch.ones(dim, device=DEV)
    data = normal(3, steps, 3, heads + 2 * kv, dim, dtype=BF16).to(DEV)

    def step(x, cache, batch, positions):
        q = attention.append(x[:, heads:heads + kv], x[:, heads + kv:], cache, batch, q=x[:, :heads], positions=positions,
                             turns=table, q_weight=w, k_weight=w)
        return attention.attend(q, cache, batch)

    def state():
        cache = attention.Cache(*(t.clone() for t in first))
        return cache, whole._replace(lengths=i32(*lengths).to(DEV)), i32(*(n - 1 for n in lengths)).to(DEV)
    cache, batch, positions = state()
    eager = []
    for i in range(steps):
        eager.append(step(data[i], cache, batch, positions).clone())
        batch.lengths.add_(1), positions.add_(1)
    kept = [t.clone() for t in cache]
    cache, batch, positions = state()
    x = data[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, cache, batch, positions)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, cache, batch, positions)
    for a, b in zip(cache, first):
        a.view(torch.int8).copy_(b.view(torch.int8))
    for i in range(steps):
        x.copy_(data[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i])
        batch.lengths.add_(1), positions.add_(1)
    assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(kept, cache))


def test_declined():
    cache = attention.new_cache(2, 1, 96, device=DEV)
    batch, _ = make_batch([3], [1], blocks=2)
    x = torch.zeros(1, 1, 96, dtype=F16, device=DEV)
    assert attention.attend(x, cache, batch) is None and attention.append(x, x, cache, batch) is None
    assert attention.read(cache, batch) is None and attention.norm_rope(x, x) is None
    cache = attention.new_cache(2, 1, 64, device=DEV)
    assert attention.attend(torch.zeros(1, 1, 64, device=DEV), cache, batch) is None


class _None:
    """Hands every call over to attention.py."""

    def __getattr__(self, name):
        return lambda *args: NotImplemented


def test_binding_and_python_calls_agree(monkeypatch):
    """The compiled calls take what fits, on the current stream, and give the bits of the calls made in Python; what does not
    fit (copies of odd strides, refusals, declines) is the same through either."""
    heads, kv, dim = 6, 2, 128
    batch, blocks = make_batch([100, 40], [2, 3], seed=4)
    first = gpu(random_cache(blocks, kv, dim, E4M3, seed=6))
    qkv = normal(3, 5, heads + 2 * kv, dim, dtype=BF16).to(DEV)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    table, positions, w = attention.turns(dim, device=DEV), i32(98, 99, 37, 38, 39).to(DEV), torch.full((dim,), 1.5, device=DEV)
    odd = torch.zeros(5, heads, dim + 1, dtype=BF16, device=DEV)[..., 1:]
    odd.copy_(q)

    def calls():
        cache = attention.Cache(*(t.clone() for t in first))
        got = [*attention.norm_rope(q, k, positions, table, w, w, interleaved=True, factor=0.5), *attention.norm_rope(q, k),
               attention.append(k, v, cache, batch, q=q, positions=positions, turns=table, q_weight=w, k_weight=w, eps=1e-5),
               attention.attend(q, cache, batch, window=9), attention.attend(odd, cache, batch, scale=1),
               attention.attend(q, cache, batch, causal=False), *attention.read(cache, batch, tail=70, dtype=F32), *attention.read(cache, batch)]
        assert attention.append(k, v, cache, batch) is True
        assert attention.attend(q.float(), cache, batch) is None
        with pytest.raises(ValueError):
            attention.attend(q[..., :64], cache, batch)
        with pytest.raises(ValueError):
            attention.norm_rope(q, k, positions[:3], table)
        return got + [t.view(INT8) if t.dtype is E4M3 else t for t in cache]

    assert attention._bind.attend(q, first, batch, None, True, 0) is not NotImplemented
    assert attention._bind.read(first, batch, None, F16) is not NotImplemented
    assert attention._bind.norm_rope(q, k, positions, table, w, w, 1e-6, False, 1.0) is not NotImplemented
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        compiled = calls()
    torch.cuda.current_stream().wait_stream(side)
    monkeypatch.setattr(attention, "_bind", _None())
    for a, b in zip(compiled, calls(), strict=True):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- sequences longer than their table
@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("lengths,rows", [([65, 130], [1, 2]), ([68, 300], [5, 290]), ([129, 64], [70, 1]), ([2 ** 31 - 1, 60], [3, 1])])
def test_tokens_past_the_table_are_written_nowhere(dtype, lengths, rows):
    """Rows stand at their own positions, also where the table ends before or among them: those past it leave what it holds
    alone, and the others go where a longer table puts them."""
    print(f"append {dtype} {lengths} {rows}", flush=True)
    table = i32(2, 5).view(2, 1).to(DEV)
    starts = [0, rows[0], sum(rows)]
    batch = attention.Batch(table, i32(*lengths).to(DEV), i32(*starts).to(DEV), max(rows), min(max(lengths), 512))
    first = gpu(random_cache(8, 2, 64, dtype))
    cache = attention.Cache(*(t.clone() for t in first))
    model = Model(first)
    k, v = normal(1, sum(rows), 2, 64) * 9, normal(2, sum(rows), 2, 64) * 9  # the partly filled blocks' scales grow
    assert attention.append(k.to(DEV), v.to(DEV), cache, batch) is True
    for which, t in enumerate((k, v)):
        for s in range(2):
            at = lengths[s] - rows[s]
            if at < 64:
                model.append(which, t[starts[s]:starts[s + 1]], [(2, 5)[s]], at)
    model.check(cache)
    for b in range(8):
        if b not in (2, 5) or lengths[(2, 5).index(b)] - rows[(2, 5).index(b)] >= 64:
            assert all(torch.equal(x[b].view(INT8), y[b].view(INT8)) for x, y in zip(cache, first))
    # read back: positions before lengths[s], zeros past the table
    tail = 80
    for got, which in zip(attention.read(cache, batch, tail=tail, dtype=F32), (0, 1)):
        for s in range(2):
            want = torch.zeros(tail, 2, 64, dtype=torch.float64)
            ref = values(cache, batch, s, 64)[which]
            for i in range(tail):
                if 0 <= lengths[s] - tail + i < 64:
                    want[i] = ref[lengths[s] - tail + i]
            assert torch.all((got[s].cpu().double() - want).abs() <= 2 * u(F32) * want.abs())


@pytest.mark.parametrize("lengths,rows,causal,window", [
    ([200, 70], [1, 1], True, 0), ([140, 66], [9, 5], True, 0), ([300, 129], [1, 2], True, 100), ([330, 200], [70, 100], True, 0),
    ([210, 140], [60, 40], True, 20), ([300, 90], [40, 3], False, 0), ([9000, 20000], [40, 1], True, 9000),
    ([2 ** 31 - 1, 128], [2, 2], True, 0), ([2 ** 31 - 1, 2 ** 31 - 1], [2, 40], False, 0)])
@pytest.mark.parametrize("heads,group,dim,dtype,x", [(2, 4, 128, INT8, BF16), (1, 2, 64, E4M3, F16), (1, 3, 256, INT8, F16)])
def test_attend_past_the_table(lengths, rows, causal, window, heads, group, dim, dtype, x):
    """Causal order and windows go by the rows' own positions where the table holds only the first 128 tokens."""
    print(f"attend {lengths} {rows} {causal} {window} {heads} x {group} x {dim} {dtype} {x}", flush=True)
    table = i32(1, 4, 0, 3).view(2, 2).to(DEV)
    batch = attention.Batch(table, i32(*lengths).to(DEV), i32(0, rows[0], sum(rows)).to(DEV), max(rows), min(max(lengths), 1 << 16))
    cache = random_cache(6, heads, dim, dtype, seed=4)
    q = normal(3, sum(rows), heads * group, dim, dtype=x)
    got = attention.attend(q.to(DEV), gpu(cache), batch, causal=causal, window=window)
    out, bound, shift = (torch.zeros(*q.shape[:2], n, dtype=torch.float64) for n in (dim, dim, 1))
    at = 0
    for s in range(2):
        for i in range(rows[s]):  # a row sees what one row at its place sees of the 128 tokens
            end = lengths[s] - rows[s] + i + 1 if causal else lengths[s]
            begin = max(end - window, 0) if window else 0
            end = min(end, 128)
            if begin < end:
                one = attention.Batch(batch.table[s:s + 1], i32(end), i32(0, 1), 1, end)
                for to, part in zip((out, bound, shift), attention_reference(q[at:at + 1], cache, one, dim ** -0.5, True, end - begin)):
                    to[at] = part[0]
            at += 1
    attention_close(got, q, (out, bound, shift))


def test_captured_steps_past_the_table():
    """A captured step that is replayed after its table is full drops the new tokens: nothing that is held changes."""
    table = i32(3, 1).view(1, 2).to(DEV)
    lengths = i32(126).to(DEV)
    batch = attention.Batch(table, lengths, i32(0, 1).to(DEV), 1, 128)
    cache = gpu(random_cache(4, 2, 128, INT8, seed=9))
    k, v = (normal(1, 1, 2, 128) * 30).to(DEV), normal(2, 1, 2, 128).to(DEV)

    def step():
        lengths.add_(1)
        attention.append(k, v, cache, batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    torch.cuda.synchronize()
    assert lengths.item() == 128
    full = [t.clone() for t in cache]
    k.mul_(50), v.mul_(50)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(cache, full))


@pytest.mark.parametrize("lengths,rows,causal,window", [([700], [3], True, 0), ([700, 300], [40, 300], True, 0), ([900], [70], True, 130),
                                                        ([333], [33], False, 0), ([20000], [1], True, 0)])
@pytest.mark.parametrize("scale", [-0.6, 0.6])
@pytest.mark.parametrize("heads,group,dim,dtype,x", [(1, 4, 128, INT8, BF16), (2, 2, 64, E4M3, F16), (1, 3, 256, INT8, F16)])
def test_attend_scales_of_either_sign(lengths, rows, causal, window, scale, heads, group, dim, dtype, x):
    """Logits of some tens: a row's reference moves as it goes, and one or a few tokens take all the weight."""
    print(f"attend {lengths} {rows} {causal} {window} {scale} {heads} x {group} x {dim} {dtype} {x}", flush=True)
    batch, blocks = make_batch(lengths, rows, seed=1)
    cache = random_cache(blocks, heads, dim, dtype, seed=sum(lengths))
    q = normal(3, sum(rows), heads * group, dim, dtype=x)
    got = attention.attend(q.to(DEV), gpu(cache), batch, scale=scale, causal=causal, window=window)
    attention_close(got, q, attention_reference(q * math.copysign(1, scale), cache, batch, abs(scale), causal, window))


@pytest.mark.parametrize("x", [F16, F32])
@pytest.mark.parametrize("rows,heads", [(1, 4), (3, 1), (1, 1)])
def test_slices_of_one_row_or_head(rows, heads, x):
    """One row of a projection whose rows are an odd step apart, one head of several that are: served as the dense tensor is."""
    batch, blocks = make_batch([70], [rows], seed=1)
    first = gpu(random_cache(blocks, heads, 64, INT8, seed=2))
    wide = normal(5, 4, 771, dtype=x).to(DEV)
    if heads > 1:
        slices = [wide[:, at:at + 64 * heads].unflatten(1, (heads, 64))[r:r + 1] for r, at in ((0, 0), (1, 0), (0, 3))]
    else:
        slices = [normal(6, 4, 5, 65, dtype=x).to(DEV)[:rows, at:at + 1, at:at + 64] for at in (0, 1)]
    for t in slices:
        dense = torch.empty(t.shape, dtype=x, device=DEV).copy_(t)
        w = torch.full((64,), 1.5, device=DEV)
        for y, z in zip(attention.norm_rope(t, t, q_weight=w), attention.norm_rope(dense, dense, q_weight=w)):
            assert torch.equal(y, z)
        pools = []
        for y in (t, dense):
            cache = attention.Cache(*(a.clone() for a in first))
            assert attention.append(y, y, cache, batch, q=y, k_weight=w) is not None
            pools.append(cache)
        assert all(torch.equal(a, b) for a, b in zip(*pools))
        if x is F16:
            got = attention.attend(t, pools[0], batch)
            assert got is not None and torch.equal(got, attention.attend(dense, pools[1], batch))


def test_norm_rope_of_more_heads_than_a_grid_is_tall():
    """Heads go over the grid's second axis in turns: 2^21 + 3 of them, one row."""
    heads = (1 << 21) + 3
    x = normal(1, 1, 8, 64, dtype=F16).to(DEV).repeat(1, heads // 8 + 1, 1)[:, :heads]
    w = torch.full((64,), 1.5, device=DEV)
    few, _ = attention.norm_rope(x[:, :8], x[:, :0], q_weight=w)
    many, _ = attention.norm_rope(x, x[:, :0], q_weight=w)
    assert torch.equal(many, few.repeat(1, heads // 8 + 1, 1)[:, :heads])


@pytest.mark.parametrize("x", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_codes_are_those_of_the_quotient(dtype, x, dim):
    """Values at the borders between codes and a step beside them: the scale is the largest by 127 or 448 and the code that of
    x by the scale, each one division in fp32, bit for bit."""
    rows, heads, m = 150, 2, LIMIT[dtype]
    batch, blocks = make_batch([rows], [rows], seed=4)
    g = torch.Generator().manual_seed(dim)
    size = 2.0 ** (torch.rand((1, heads, 1), generator=g) * 40 - 20)
    code = torch.arange(127, dtype=INT8)
    code = code.float() if dtype is INT8 else code.view(E4M3).float()
    grid = (code[1:] + code[:-1]) / 2
    grid = torch.cat((-grid, grid))
    new = []
    for _ in range(2):
        t = grid[torch.randint(len(grid), (rows, heads, dim), generator=g)] / m * size
        t[0::64, :, 0] = size[0, :, 0]  # each block's largest
        t = torch.nextafter(t, t * torch.tensor([0.0, 1.0, 4.0])[torch.randint(3, t.shape, generator=g)])
        new.append(torch.minimum(t.abs(), size).copysign(t).to(x))
    cache = gpu(random_cache(blocks, heads, dim, dtype))
    assert attention.append(*(t.to(DEV) for t in new), cache, batch) is True
    for t, codes, scales, turned in ((new[0], cache.k, cache.k_scale, False), (new[1], cache.v, cache.v_scale, True)):
        for j, b in enumerate(batch.table[0].tolist()):
            part = t[64 * j:64 * j + 64].float().transpose(0, 1)
            scale = part.abs().amax((1, 2)) / m
            assert torch.equal(scales[b].cpu(), scale)
            want = (part / scale[:, None, None]).clamp(-m, m)
            want = (want.round() if dtype is INT8 else want).to(dtype)
            got = codes[b].cpu().view(INT8)
            got = (got.transpose(-1, -2) if turned else got)[:, :part.shape[1]]
            assert torch.equal(got, want.view(INT8))


@pytest.mark.parametrize("n,heads,group,dim,length,rows,window", [
    (16, 4, 8, 128, 300, 256, 0), (16, 4, 8, 128, 700, 256, 130), (24, 2, 2, 64, 8200, 260, 0), (24, 2, 2, 64, 8200, 260, 5000),
    (24, 2, 2, 64, 8200, 260, 900)])
@pytest.mark.parametrize("dtype,x", [(INT8, BF16), (E4M3, F16)])
@pytest.mark.parametrize("scale", [None, 0.6])
def test_attend_many_tiles(n, heads, group, dim, length, rows, window, dtype, x, scale):
    """So many rows that no call is split: 256 rows a workgroup for heads of 128, and of 64 over long caches or wide windows,
    128 else. All sequences but one have the same blocks."""
    print(f"attend {n} x {rows} over {length} window {window} {heads} x {group} x {dim} {dtype} {x} {scale}", flush=True)
    batch, blocks = make_batch([length, length], [rows, rows], seed=1)
    cache = random_cache(blocks, heads, dim, dtype, seed=7)
    order = [0] * (n - 1) + [1]
    ragged = [rows - (s * 7) % 64 for s in range(n)]
    starts = i32(0, *torch.tensor(ragged).cumsum(0).tolist())
    lengths = i32(*(length - s for s in range(n)))
    many = attention.Batch(batch.table[order].contiguous(), lengths.to(DEV), starts.to(DEV), rows, length)
    q = normal(3, sum(ragged), heads * group, dim, dtype=x)
    got = attention.attend(q.to(DEV), gpu(cache), many, scale=scale, window=window)
    for s in (0, n // 2, n - 1):
        one = attention.Batch(many.table[s:s + 1], lengths[s:s + 1], i32(0, ragged[s]), rows, length)
        part = slice(int(starts[s]), int(starts[s + 1]))
        attention_close(got[part], q[part], attention_reference(q[part], cache, one, dim ** -0.5 if scale is None else scale, True, window))


def test_append_of_many_rows_with_queries():
    """Above 2048 rows a wave turns a row's queries by itself."""
    rows, lengths, heads, kv, dim = [1500, 600], [1530, 600], 6, 2, 64
    batch, blocks = make_batch(lengths, rows, seed=3)
    cache = random_cache(blocks, kv, dim, INT8, seed=8)
    model, cache = Model(cache), gpu(cache)
    qkv = normal(5, sum(rows), heads + 2 * kv, dim, dtype=BF16)
    positions = torch.cat([torch.arange(n - r, n) for n, r in zip(lengths, rows)]).int()
    inv = [1e4 ** (-2.0 * i / dim) for i in range(dim // 2)]
    wq, wk = 1 + normal(2, dim) / 4, 2 + normal(3, dim) / 4
    d = qkv.to(DEV)
    q = attention.append(d[:, heads:heads + kv], d[:, heads + kv:], cache, batch, q=d[:, :heads], positions=positions.to(DEV),
                         turns=attention.turns(inv_freq=inv, device=DEV), q_weight=wq.to(DEV), k_weight=wk.to(DEV))
    y = rope_reference(qkv[:, :heads], positions, inv, wq, 1e-6, False)
    assert torch.all((q.cpu().double() - y).abs() <= rope_tolerance(y, qkv[:, :heads], wq, 1e-6, BF16))
    k = rope_reference(qkv[:, heads:heads + kv], positions, inv, wk, 1e-6, False)
    for s, part in enumerate((slice(0, 1500), slice(1500, 2100))):
        for which, t in enumerate((k, qkv[:, heads + kv:])):
            model.append(which, t[part], batch.table[s].tolist(), lengths[s] - rows[s])
    model.check(cache, key_error=2.0 ** -18)  # see rope_tolerance: 2^-19 sqrt 2 of the head's largest


@pytest.mark.parametrize("rows", [2, 80])
def test_attend_queries_of_subnormal_values(rows):
    """bf16 queries down to 2^-133: logits of next to nothing, so that every token seen has the same weight."""
    batch, blocks = make_batch([200], [rows], seed=1)
    cache = random_cache(blocks, 2, 128, INT8, seed=5)
    q = (normal(3, rows, 4, 128) * 2.0 ** -131).to(BF16)
    q[0] = 0
    got = attention.attend(q.to(DEV), gpu(cache), batch)
    attention_close(got, q, attention_reference(q, cache, batch, 128 ** -0.5, True, 0))
