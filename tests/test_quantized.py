"""The cache held in 8 bits: rows written as codes and scales, pages read back, and the decode attention over the codes,
each against its definition in 64 bits."""
import math

import pytest
import torch

LIMITS = {"fp8": 448.0, "int8": 127.0}
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}    # a rounding's half step, relative to the value

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from metallix_b200 import ops
    ops.require_cuda()
    return ops


def nearest_code(y, kind):
    """The code nearest to y (float64), halves to the even one, as the number it stands for."""
    if kind == "int8":
        return y.round().clamp(-127, 127)
    y = y.clamp(-448.0, 448.0)
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y).exponent.clamp(min=-5) - 4)
    return (y / step).round() * step


def exact_rows(x, kind):
    """(scale, code values) of rows x [..., head_dim] of float32 or bfloat16 numbers, in 64 bits; the scale as float32 holds it."""
    x = x.double()
    scale = (x.abs().amax(-1).float() / torch.full((), LIMITS[kind], device=x.device)).double()
    y = x / torch.where(scale > 0, scale, 1.0).unsqueeze(-1)
    return scale, nearest_code(y, kind)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def spread_tables(lengths, page, seed, spare=2):
    """Block tables whose pages lie anywhere in the pool: (pages of the pool, tables [requests, width])."""
    counts = [-(-n // page) for n in lengths]
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(counts) + spare, generator=gen).tolist()
    table = torch.full((len(lengths), max(max(counts), 1)), -1, dtype=torch.int32)
    for row, count in enumerate(counts):
        for i in range(count):
            table[row, i] = order.pop()
    return sum(counts) + spare, table.cuda()


def random_pool(ops, kind, pages, kv_heads, page, head_dim, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pool = ops.QuantizedPool.zeros(pages, kv_heads, page, head_dim, codes=kind)
    x = torch.randn(pool.shape, generator=gen, device="cuda")
    scale, codes = exact_rows(x, kind)
    pool.codes.copy_(codes.to(pool.codes.dtype))
    pool.scales.copy_(scale)
    return pool


def values_of(pool):
    """What the pool stands for, in float64."""
    return pool.codes.float().double() * pool.scales.double().unsqueeze(-1)


# ----------------------------------------------------------------- refusals, without a GPU
def test_a_pool_says_what_is_wrong_with_it():
    from metallix_b200 import ops
    codes, scales = torch.zeros(3, 2, 1, 4, 8, dtype=torch.int8), torch.zeros(3, 2, 1, 4)
    with pytest.raises(ops.KernelError, match="CUDA device"):
        ops.QuantizedPool(codes, scales)
    with pytest.raises(ops.KernelError, match="codes must be one of"):
        ops.QuantizedPool.zeros(3, 1, 4, 8, codes="int4")
    with pytest.raises(ops.KernelError, match="QuantizedPool"):
        ops.read_cache(codes, codes, None, None, None, None)


# ----------------------------------------------------------------- the write
@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim,kv_heads,page,tokens", [(128, 2, 16, 37), (64, 5, 8, 33), (256, 1, 32, 9), (48, 3, 4, 21), (20, 2, 1, 6),
                                                           (128, 8, 16, 1)])
def test_rows_written_are_the_nearest_codes(ops, kind, dtype, head_dim, kv_heads, page, tokens):
    """Keys and values as they are: scales and codes have one right answer each, bit for bit."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    wide = torch.randn((tokens, 3 * kv_heads * head_dim + 16), generator=gen, device="cuda").to(dtype)
    k = wide[:, 8:8 + kv_heads * head_dim]               # rows of a wider product
    v = wide[:, 8 + kv_heads * head_dim:8 + 2 * kv_heads * head_dim]
    pages = -(-tokens // page) + 2
    pool = random_pool(ops, kind, pages, kv_heads, page, head_dim, 3)
    before_codes, before_scales = pool.codes.clone(), pool.scales.clone()
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:tokens].to(torch.int32)
    if tokens > 5:
        slots[4] = -1      # a token that is not written
    ops.write_cache(k, v, pool, slots.cuda(), ints([0] * tokens))
    ops.check_status("cuda")
    written = slots.tolist()
    for plane, rows in enumerate((k, v)):
        scale, codes = exact_rows(rows.reshape(tokens, kv_heads, head_dim), kind)
        for t, slot in enumerate(written):
            if slot < 0:
                continue
            at = (slot // page, plane, slice(None), slot % page)
            assert torch.equal(pool.scales[at].double(), scale[t])
            assert torch.equal(pool.codes[at].float().double(), codes[t])
            before_codes[at], before_scales[at] = pool.codes[at], pool.scales[at]
    # everything else is as it was
    assert torch.equal(pool.codes.view(torch.uint8), before_codes.view(torch.uint8)) and torch.equal(pool.scales, before_scales)


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("head_dim", [128, 48])
def test_quotients_next_to_the_middle_of_two_codes(ops, kind, head_dim):
    """Numbers an ulp to either side of, and on, the middle between two codes, at scales from 2^-140 to 2^118."""
    gen = torch.Generator().manual_seed(7)
    rows = []
    for exponent in (-140, -127, -100, -61, -60, -3, 0, 5, 59, 61, 100, 118):
        for mantissa in (1.0, 1.0 + 2.0 ** -23, 1.37, 2.0 - 2.0 ** -23):
            top = torch.tensor(mantissa * 2.0 ** exponent, dtype=F32)
            scale = top / LIMITS[kind]
            values = torch.arange(-126, 127).double() + 0.5 if kind == "int8" else \
                torch.tensor([(8 + i + 0.5) * 2.0 ** (e - 3) for i in range(8) for e in range(-6, 8)] + [(i + 0.5) * 2.0 ** -9 for i in range(8)]).double()
            middle = values[torch.randint(len(values), (head_dim - 1,), generator=gen)] * scale.double()
            x = middle.float()
            step = torch.randint(-1, 2, (head_dim - 1,), generator=gen)
            x = torch.where(step > 0, torch.nextafter(x, torch.tensor(math.inf)), torch.where(step < 0, torch.nextafter(x, torch.tensor(-math.inf)), x))
            rows.append(torch.cat([top.reshape(1), x.clamp(-top, top)]))
    k = torch.stack(rows).cuda()
    tokens = k.shape[0]
    pool = ops.QuantizedPool.zeros(tokens, 1, 1, head_dim, codes=kind)
    ops.write_cache(k, -k, pool, ints(list(range(tokens))), ints([0] * tokens))
    for plane, x in enumerate((k, -k)):
        scale, codes = exact_rows(x, kind)
        assert torch.equal(pool.scales[:, plane, 0, 0].double(), scale)
        assert torch.equal(pool.codes[:, plane, 0, 0].float().double(), codes)


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("head_dim", [64, 20])
def test_rows_of_zeros_and_rows_that_are_not_finite(ops, kind, head_dim):
    k = torch.ones(5, head_dim, device="cuda")
    k[0] = 0.0
    k[1, 3] = math.inf
    k[2, head_dim - 1] = math.nan
    k[3, 0] = -math.inf
    k[4] = 1e-45          # the smallest number there is
    pool = ops.QuantizedPool.zeros(5, 1, 1, head_dim, codes=kind)
    pool.codes.view(torch.uint8).fill_(0x11)
    ops.write_cache(k, k, pool, ints(range(5)), ints([0] * 5))
    assert pool.scales[0].eq(0).all() and pool.scales[1:4].isnan().all()
    out = torch.full(pool.shape, 7.0, device="cuda")
    ops.read_cache(pool, out, ints([[0], [1], [2], [3], [4]]), ints(range(5)), ints([0] * 5), ints([0] * 5))
    assert out[0].eq(0).all() and out[1:4].isnan().all() and out[4].isfinite().all()
    ops.check_status("cuda")


def turned(x, cos, sin, positions, interleaved):
    """Rotation of [tokens, heads, head_dim] in float64."""
    half = cos.shape[1]
    where = torch.arange(half, device=x.device)
    i, j = (2 * where, 2 * where + 1) if interleaved else (where, where + half)
    c, s = cos.double()[positions.long()].unsqueeze(1), sin.double()[positions.long()].unsqueeze(1)
    out = x.clone()
    out[..., i] = x[..., i] * c - x[..., j] * s
    out[..., j] = x[..., j] * c + x[..., i] * s
    return out


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim,heads,kv_heads,rotary,interleaved,scope,tokens", [
    (128, 4, 2, 128, False, "head", 19), (64, 6, 2, 64, True, "head", 7), (128, 8, 4, 64, False, "head", 40),
    (256, 2, 1, 256, False, "head", 5), (48, 3, 1, 24, False, "head", 11), (128, 4, 2, 128, False, "projection", 6),
    (20, 4, 2, 12, True, "projection", 5), (64, 4, 4, 0, False, "head", 9), (128, 16, 8, 128, False, None, 3),
    (256, 4, 4, 64, True, None, 13), (128, 32, 8, 128, False, "head", 700), (64, 15, 5, 64, True, None, 900)])
def test_norm_rotation_and_write(ops, kind, dtype, head_dim, heads, kv_heads, rotary, interleaved, scope, tokens):
    """Queries as the write into a cache of the compute type gives them; keys: a code is the nearest one to the quotient, but
    for what the row's own rounding in 32 bits moves it by."""
    gen = torch.Generator(device="cuda").manual_seed(head_dim + tokens)
    width = (heads + 2 * kv_heads) * head_dim
    qkv = torch.randn((tokens, width), generator=gen, device="cuda").to(dtype)
    q, k, v = qkv.split([heads * head_dim, kv_heads * head_dim, kv_heads * head_dim], 1)
    positions = torch.randint(0, 300, (tokens,), generator=gen, device="cuda").to(torch.int32)
    page, pages = 8, -(-tokens // 8) + 1
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(5))[:tokens].to(torch.int32).cuda()
    weight = lambda n: 1.0 + 0.2 * torch.randn(n, generator=gen, device="cuda")  # noqa: E731
    whole = scope == "projection"
    qw, kw = (weight(heads * head_dim if whole else head_dim), weight(kv_heads * head_dim if whole else head_dim)) if scope else (None, None)
    cos = sin = None
    if rotary:
        angle = torch.rand((300, rotary // 2), generator=gen, device="cuda") * 6.28
        cos, sin = angle.cos(), angle.sin()
    factors = 0.5 + torch.rand(300, generator=gen, device="cuda")
    pool = ops.QuantizedPool.zeros(pages, kv_heads, page, head_dim, codes=kind)
    plain = torch.zeros(pool.shape, dtype=dtype, device="cuda")
    outs = [torch.zeros((tokens, heads, head_dim), dtype=dtype, device="cuda") for _ in range(2)]
    for cache, out in zip((pool, plain), outs):
        ops.qk_norm_rope_cache(q, k, v, out, cache, slots, positions, qw, kw, cos, sin, 1e-6, interleaved=interleaved,
                               norm_scope=scope or "head", q_factors=factors)
    ops.check_status("cuda")

    def exact(x, w):
        x = x.double().reshape(tokens, -1, head_dim)
        if w is not None:
            mean = x.square().mean((1, 2), keepdim=True) if whole else x.square().mean(-1, keepdim=True)
            x = x * torch.rsqrt(mean + 1e-6) * (w.double().view(-1, head_dim) if whole else w.double())
        return turned(x, cos, sin, positions, interleaved) if rotary else x

    # a value in 32 bits: the row's sum of squares and root, two products, and a rotation of two more products and a sum
    bits = 16 * 2.0 ** -24
    query = exact(q, qw) * factors.double()[positions.long()][:, None, None]
    size = query.abs().amax(-1, keepdim=True)
    for out in outs:
        assert ((out.double() - query).abs() <= HALF[dtype] * query.abs() + bits * 1.5 * size).all()
    held, row = slots.long() // page, slots.long() % page
    key = exact(k, kw)
    scale = pool.scales[held, 0, :, row].double()
    size = key.abs().amax(-1)
    assert ((scale * LIMITS[kind] - size).abs() <= 2 * bits * size).all()
    code = pool.codes[held, 0, :, row].float().double()
    y = key / scale.unsqueeze(-1)
    off = (code - y).abs()
    best = (nearest_code(y, kind) - y).abs()
    assert (off <= best + 2 * 2 * bits * LIMITS[kind]).all()      # another code only where both are as near
    value_scale, value_codes = exact_rows(v.reshape(tokens, kv_heads, head_dim), kind)
    assert torch.equal(pool.scales[held, 1, :, row].double(), value_scale)
    assert torch.equal(pool.codes[held, 1, :, row].float().double(), value_codes)


@gpu
def test_a_slot_or_position_outside_its_table_is_reported(ops):
    pool = ops.QuantizedPool.zeros(2, 1, 4, 64)
    k = torch.ones(2, 64, device="cuda", dtype=BF16)
    ops.write_cache(k, k, pool, ints([8, 0]), ints([0, 0]))
    with pytest.raises(ops.KernelError, match="slot or position"):
        ops.check_status("cuda")
    assert pool.scales[0, 0, 0, 0] > 0 and pool.scales.count_nonzero() == 2
    cos = torch.ones(4, 32, device="cuda")
    ops.qk_norm_rope_cache(k[:, :0], k, k, None, pool, ints([1, 2]), ints([4, -1]), None, None, cos, cos, 0.0)
    with pytest.raises(ops.KernelError, match="slot or position"):
        ops.check_status("cuda")


@gpu
def test_refusals_of_the_write(ops):
    pool = ops.QuantizedPool.zeros(2, 1, 4, 64)
    k = torch.ones(2, 64, device="cuda", dtype=BF16)
    with pytest.raises(ops.KernelError, match="widths"):
        ops.write_cache(k[:, :32], k[:, :32], pool, ints([0, 1]), ints([0, 0]))
    with pytest.raises(ops.KernelError, match="one slot per token"):
        ops.write_cache(k, k, pool, ints([0]), ints([0, 0]))
    with pytest.raises(ops.KernelError, match="one scale per row"):
        ops.QuantizedPool(pool.codes, pool.scales[:, :1].contiguous())
    with pytest.raises(ops.KernelError, match="dtype"):
        ops.QuantizedPool(pool.codes.view(torch.uint8), pool.scales)
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.QuantizedPool(pool.codes.transpose(3, 4), pool.scales)


# ----------------------------------------------------------------- reading back
@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim,kv_heads,page", [(128, 2, 16), (64, 3, 8), (256, 1, 64), (40, 2, 4), (24, 1, 1), (13, 2, 2)])
@pytest.mark.parametrize("window,chunk,keep", [(0, 0, 0), (9, 0, 0), (0, 32, 0), (20, 0, 6)])
def test_pages_read_back(ops, kind, dtype, head_dim, kv_heads, page, window, chunk, keep):
    lengths = [1, 50, 0, 77, 16, 33]
    firsts = [0, 45, 0, 40, 15, 0]
    pages, table = spread_tables(lengths, page, 2)
    pool = random_pool(ops, kind, pages, kv_heads, page, head_dim, 4)
    order = [3, 0, 5, 1, 4, 2]
    out = torch.full(pool.shape, 7.0, dtype=dtype, device="cuda")
    ops.read_cache(pool, out, table, ints(order), ints([firsts[r] for r in order]), ints([lengths[r] - 1 for r in order]),
                   window=window, chunk=chunk, keep=keep)
    ops.check_status("cuda")
    expect = torch.full(pool.shape, 7.0, dtype=dtype, device="cuda")
    values = (pool.codes.float() * pool.scales.unsqueeze(-1)).to(dtype)
    for r, length in enumerate(lengths):
        begin = max(firsts[r] - window + 1, 0) if window else 0
        if chunk:
            begin = max(begin, firsts[r] - firsts[r] % chunk)
        for slot in range(-(-length // page)):
            if (slot + 1) * page <= begin and slot * page >= keep:
                continue
            at, rows = int(table[r, slot]), min(page, length - slot * page)
            expect[at, :, :, :rows] = values[at, :, :, :rows]
    assert torch.equal(out, expect)


@gpu
def test_a_page_outside_the_pool_is_reported_and_not_read(ops):
    pool = random_pool(ops, "fp8", 3, 1, 4, 64, 0)
    out = torch.zeros(pool.shape, device="cuda")
    ops.read_cache(pool, out, ints([[1, 3, -1]]), ints([0]), ints([0]), ints([11]))
    with pytest.raises(ops.KernelError, match="block-table"):
        ops.check_status("cuda")
    assert out[1].abs().sum() > 0 and out[0].eq(0).all() and out[2].eq(0).all()
    with pytest.raises(ops.KernelError, match="pool's shape"):
        ops.read_cache(pool, out[:2], ints([[1]]), ints([0]), ints([0]), ints([3]))
    with pytest.raises(ops.KernelError, match="differ in length"):
        ops.read_cache(pool, out, ints([[1]]), ints([0]), ints([0, 0]), ints([3]))


# ----------------------------------------------------------------- the decode attention
def exact_decode(q, pool, table, rows, positions, scale, window=0, chunk=0, keep=0, softcap=0.0, sink=None, bias=None, gate=None):
    """(out, bound) [tokens, heads, head_dim] in float64 of the rows (token, request): what comes out, and the sum of the
    weights times the values' magnitudes, which roundings of the weights are relative to."""
    values = values_of(pool)
    page, kv_heads = pool.shape[3], pool.shape[2]
    tokens, heads, head_dim = q.shape
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for token, request in rows:
        pos = int(positions[token])
        at = torch.arange(pos + 1)
        first = max(pos - window + 1, 0) if window else 0
        if chunk:
            first = max(first, pos - pos % chunk)
        at = at[(at >= first) | (at < keep)]
        held, row = table[request].cpu().long()[at // page].cuda(), (at % page).cuda()
        keys, vals = (values[held, plane, :, row].repeat_interleave(heads // kv_heads, 1) for plane in (0, 1))
        s = torch.einsum("hd,khd->hk", q[token].double(), keys) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if bias is not None:
            s = s + bias.double()[:, (pos - at).clamp(max=bias.shape[1] - 1).cuda()]
        if sink is not None:
            extra = sink.double() if isinstance(sink, torch.Tensor) else torch.full((heads,), sink, dtype=torch.float64, device="cuda")
            s = torch.cat([s, extra[:, None]], 1)
        p = torch.softmax(s, 1)[:, :len(at)]
        out[token] = torch.einsum("hk,khd->hd", p, vals)
        bound[token] = torch.einsum("hk,khd->hd", p, vals.abs())
        if gate is not None:
            g = torch.sigmoid(gate[token].double().view(heads, head_dim))
            out[token] *= g
            bound[token] *= g
    return out, bound


def close(out, exact, bound, dtype):
    """Weights in bfloat16 (in its type alone), the output's own rounding, and what a score's rounding in 32 bits does to
    its exponential: scores of up to some 30, sums of up to 256 products, 2^-24 each, three roundings of the sums."""
    per_weight = (HALF[BF16] if dtype == BF16 else 0.0) + 30 * 8 * 2.0 ** -24
    off = (out.double() - exact).abs()
    limit = per_weight * bound + HALF[dtype] * exact.abs() * 1.01 + 1e-30
    assert (off <= limit).all(), f"{(off / limit).max().item():.2f} times the bound"


SHAPES = [(128, 2, 2, 16), (128, 8, 1, 16), (64, 14, 2, 32), (128, 15, 3, 8), (256, 4, 2, 16), (64, 4, 4, 4), (64, 3, 3, 1), (128, 6, 1, 256),
          (48, 6, 2, 16), (20, 3, 1, 8), (128, 24, 2, 64), (256, 8, 1, 2)]


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim,heads,kv_heads,page", SHAPES)
@pytest.mark.parametrize("lengths", [[1], [2, 129, 128, 127], [700, 1, 33, 2500], [5000, 4097]])
def test_decode(ops, kind, dtype, head_dim, heads, kv_heads, page, lengths):
    pages, table = spread_tables(lengths, page, 1)
    pool = random_pool(ops, kind, pages, kv_heads, page, head_dim, 2)
    # what lies behind a request's last position, and on pages that nobody holds, is no number
    for r, n in enumerate(lengths):
        if n % page:
            pool.scales[int(table[r, n // page]), :, :, n % page:] = math.nan
    held = set(table[table >= 0].flatten().tolist())
    for free in set(range(pages)) - held:
        pool.scales[free] = math.inf
        pool.codes.view(torch.uint8)[free] = 0x7f
    gen = torch.Generator(device="cuda").manual_seed(9)
    n = len(lengths)
    q = torch.randn((n + 2, heads, head_dim), generator=gen, device="cuda").to(dtype)
    positions = torch.zeros(n + 2, dtype=torch.int32, device="cuda")
    tokens = [(3 * r + 1) % (n + 2) if math.gcd(3, n + 2) == 1 else r for r in range(n)]
    rows = list(zip(tokens, range(n)))
    for token, r in rows:
        positions[token] = lengths[r] - 1
    out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
    scale = 1.0 / math.sqrt(head_dim)
    got = ops.paged_attention_decode(q, pool, out, table, ints([rows[0][0], -1] + [t for t, _ in rows[1:]]),
                                     ints([0, 0] + list(range(1, n))), positions, scale, max(lengths))
    ops.check_status("cuda")
    assert got is out
    exact, bound = exact_decode(q, pool, table, rows, positions, scale)
    close(out[tokens], exact[tokens], bound[tokens], dtype)
    others = [t for t in range(n + 2) if t not in tokens]
    assert out[others].eq(5.0).all()      # tokens that no row names


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim,heads,kv_heads,page", [(128, 8, 2, 16), (64, 7, 1, 8), (256, 4, 2, 32), (40, 4, 2, 4)])
@pytest.mark.parametrize("options", [dict(window=1), dict(window=300), dict(chunk=256), dict(window=100, keep=5), dict(window=130, keep=200),
                                     dict(softcap=3.0), dict(sink=0.5), dict(sink="heads"), dict(bias=64), dict(gate=True),
                                     dict(window=64, softcap=5.0, sink="heads", bias=3, gate=True, keep=1)],
                         ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()))
def test_decode_options(ops, dtype, head_dim, heads, kv_heads, page, options):
    lengths = [900, 3, 257, 1500, 128]
    pages, table = spread_tables(lengths, page, 3)
    pool = random_pool(ops, "fp8", pages, kv_heads, page, head_dim, 6)
    gen = torch.Generator(device="cuda").manual_seed(1)
    n = len(lengths)
    q = torch.randn((n, heads, head_dim), generator=gen, device="cuda").to(dtype)
    positions = ints([x - 1 for x in lengths])
    options = dict(options)
    if options.get("sink") == "heads":
        options["sink"] = torch.randn(heads, generator=gen, device="cuda")
    if "bias" in options:
        options["bias"] = torch.randn((heads, options["bias"] + 1), generator=gen, device="cuda")
    if options.get("gate"):
        options["gate"] = torch.randn((n, 2 * heads * head_dim), generator=gen, device="cuda").to(dtype)[:, :heads * head_dim]
    if options.get("window"):      # pages ahead of the window have left the table, but for those that are kept
        for r, length in enumerate(lengths):
            for slot in range(max(length - options["window"], 0) // page):
                if slot * page >= options.get("keep", 0):
                    table[r, slot] = -1
    out = torch.zeros_like(q)
    scale = 1.0 / math.sqrt(head_dim)
    ops.paged_attention_decode(q, pool, out, table, ints(range(n)), ints(range(n)), positions, scale, 1500, **options)
    ops.check_status("cuda")
    exact, bound = exact_decode(q, pool, table, [(r, r) for r in range(n)], positions, scale, **options)
    if options.get("gate") is not None:      # the gate's own exponential and product
        bound = bound * (1 + 1e-4)
    close(out, exact, bound, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim,heads,kv_heads,page,rows,longest", [
    (128, 8, 4, 16, 45, 2500), (64, 12, 4, 32, 120, 1100), (256, 4, 4, 16, 30, 3000), (128, 24, 2, 8, 70, 1500), (64, 8, 8, 64, 200, 1025),
    (128, 4, 4, 16, 520, 1100), (128, 8, 8, 16, 9, 40000)])
@pytest.mark.parametrize("options", [dict(), dict(window=900, softcap=4.0, sink="heads", keep=130, gate=True)],
                         ids=["bare", "options"])
def test_decode_of_many_rows(ops, dtype, head_dim, heads, kv_heads, page, rows, longest, options):
    """Batches of many pairs, in one round of blocks and in several: contexts from one position to the longest in any order, padding rows
    between, one row beyond the bound on the contexts."""
    rng = torch.Generator().manual_seed(rows)
    lengths = torch.randint(1, longest + 1, (rows,), generator=rng).tolist()
    lengths[rows // 2], lengths[1], lengths[2] = longest, 1, 128
    pages, table = spread_tables(lengths, page, 5)
    pool = random_pool(ops, "int8" if head_dim == 64 else "fp8", pages, kv_heads, page, head_dim, 6)
    gen = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn((rows + 1, heads, head_dim), generator=gen, device="cuda").to(dtype)
    positions = ints([n - 1 for n in lengths] + [longest + 300])
    options = dict(options)
    if options.get("sink") == "heads":
        options["sink"] = torch.randn(heads, generator=gen, device="cuda")
    if options.get("gate"):
        options["gate"] = torch.randn((rows + 1, heads * head_dim), generator=gen, device="cuda").to(dtype)
    order = torch.randperm(rows, generator=rng).tolist()
    listed = [(t, t) for t in order]
    for at in (0, rows // 3, len(listed)):
        listed.insert(at, (-1, 0))
    listed.insert(rows // 4, (rows, 0))       # beyond the bound: left as it is, and reported
    out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
    scale = 1.0 / math.sqrt(head_dim)
    for _ in range(2):
        ops.paged_attention_decode(q, pool, out, table, ints([t for t, _ in listed]), ints([r for _, r in listed]), positions, scale,
                                   longest, **options)
    with pytest.raises(ops.KernelError, match="position"):
        ops.check_status("cuda")
    assert out[rows].eq(5.0).all()
    some = list(range(rows)) if rows * longest < 200_000 else sorted({1, 2, rows // 2, 0, rows - 1, rows // 5, rows // 7})
    exact, bound = exact_decode(q, pool, table, [(t, t) for t in some], positions, scale, **options)
    if options.get("gate") is not None:
        bound = bound * (1 + 1e-4)
    close(out[some], exact[some], bound[some], dtype)
    assert out[:rows].isfinite().all()


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("head_dim,heads,kv_heads", [(128, 8, 2), (64, 7, 1)])
def test_decode_with_the_output_projection(ops, kind, head_dim, heads, kv_heads):
    lengths, hidden = [900, 3, 257], 200
    pages, table = spread_tables(lengths, 16, 3)
    pool = random_pool(ops, kind, pages, kv_heads, 16, head_dim, 6)
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((4, heads, head_dim), generator=gen, device="cuda").to(BF16)
    w = (0.05 * torch.randn((hidden, heads * head_dim), generator=gen, device="cuda")).to(BF16)
    positions, scale = ints([899, 2, 256, 0]), 1.0 / math.sqrt(head_dim)
    arguments = (table, ints([0, 1, 2, -1]), ints([0, 1, 2, 0]), positions, scale, 900)
    out = torch.zeros_like(q)
    ops.paged_attention_decode(q, pool, out, *arguments)
    summands = ops.paged_attention_decode_project(q, pool, *arguments, w)
    ops.check_status("cuda")
    assert summands.shape == (heads, 4, hidden) and summands[:, 3].eq(0).all()
    parts = torch.einsum("thd,nhd->htn", out.double(), w.double().view(hidden, heads, head_dim))
    size = torch.einsum("thd,nhd->htn", out.double().abs(), w.double().abs().view(hidden, heads, head_dim))
    assert ((summands.double() - parts).abs() <= head_dim * 2.0 ** -24 * 4 * size + 1e-30).all()


@gpu
def test_decode_of_rows_that_are_not_finite_shows_it(ops):
    pool = random_pool(ops, "fp8", 2, 2, 16, 128, 0)
    pool.scales[0, 1, 1, 3] = math.nan      # a value of the second key/value head
    q = torch.ones(1, 4, 128, device="cuda", dtype=BF16)
    out = torch.zeros_like(q)
    ops.paged_attention_decode(q, pool, out, ints([[0, 1]]), ints([0]), ints([0]), ints([19]), 0.1, 20)
    assert out[0, 2:].isnan().all() and out[0, :2].isfinite().all()


@gpu
def test_decode_reports_pages_and_contexts_beyond_their_bounds(ops):
    pool = random_pool(ops, "int8", 2, 1, 16, 64, 0)
    q = torch.ones(1, 2, 64, device="cuda", dtype=BF16)
    out = torch.zeros_like(q)
    for table in ([[0, 2]], [[0, -1]], [[0]]):
        ops.paged_attention_decode(q, pool, out, ints(table), ints([0]), ints([0]), ints([19]), 0.1, 20)
        with pytest.raises(ops.KernelError, match="block-table"):
            ops.check_status("cuda")
    big = random_pool(ops, "int8", 10, 1, 16, 64, 0)
    out.fill_(3.0)
    ops.paged_attention_decode(q, big, out, ints([list(range(10))]), ints([0]), ints([0]), ints([150]), 0.1, 128)
    with pytest.raises(ops.KernelError, match="position"):
        ops.check_status("cuda")
    assert out.eq(3.0).all()


@gpu
def test_refusals_of_the_decode_attention(ops):
    pool = random_pool(ops, "fp8", 2, 2, 16, 64, 0)
    q = torch.ones(1, 4, 64, device="cuda", dtype=BF16)
    lists = (ints([[0, 1]]), ints([0]), ints([0]), ints([3]), 0.1, 20)
    with pytest.raises(ops.KernelError, match="64 values wide"):
        ops.paged_attention_decode(q[..., :32].contiguous(), pool, q[..., :32].contiguous(), *lists)
    with pytest.raises(ops.KernelError, match="does not take"):
        ops.paged_attention_decode(q[:, :3].contiguous(), pool, torch.zeros_like(q[:, :3]), *lists)
    with pytest.raises(ops.KernelError, match="negative"):
        ops.paged_attention_decode(q, pool, torch.zeros_like(q), *lists, softcap=-1.0)
    with pytest.raises(ops.KernelError, match="partial holds"):
        ops.paged_attention_decode(q, pool, torch.zeros_like(q), *lists, partial=torch.zeros(8, device="cuda"))
    with pytest.raises(ops.KernelError, match="row lists"):
        ops.paged_attention_decode(q, pool, torch.zeros_like(q), ints([[0, 1]]), ints([0]), ints([0, 0]), ints([3]), 0.1, 20)
    for other in (ops.paged_attention_tile, ops.flash_prefill):      # the kernels that read a cache of the compute type say so
        with pytest.raises(ops.KernelError, match="cache must be a tensor"):
            other(q, pool, torch.zeros_like(q), ints([[0, 1]]), ints([0]), ints([0]), ints([1]), ints([3]), 0.1)


# ----------------------------------------------------------------- numbers and calls at the edges
@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("head_dim", [64, 128, 256, 40])
def test_every_code_stands_for_its_number(ops, kind, head_dim):
    """A context of one position gives its value back: every code, through the attention and through reading back."""
    numbers = torch.arange(-127, 128).double() if kind == "int8" else \
        torch.tensor([b for b in range(256) if b & 0x7f != 0x7f], dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    rows = -(-len(numbers) // head_dim)
    values = torch.zeros(rows * head_dim, dtype=torch.float64)
    values[:len(numbers)] = numbers
    pool = ops.QuantizedPool.zeros(rows, 1, 8, head_dim, codes=kind)
    pool.codes[:, 1, 0, 0] = values.view(rows, head_dim).to(pool.codes.dtype).cuda()
    pool.scales[:, 1, 0, 0] = 2.0 ** -5
    expect = (values.view(rows, 1, head_dim) * 2.0 ** -5).float().cuda()
    for dtype in (F32, BF16):      # all of them have few enough bits for either type
        q, out = (torch.ones(rows, 1, head_dim, device="cuda", dtype=dtype) for _ in range(2))
        ops.paged_attention_decode(q, pool, out, ints([[r] for r in range(rows)]), ints(range(rows)), ints(range(rows)), ints([0] * rows),
                                   0.1, 1)
        assert torch.equal(out.float(), expect)
        back = torch.zeros(pool.shape, dtype=dtype, device="cuda")
        ops.read_cache(pool, back, ints([[r] for r in range(rows)]), ints(range(rows)), ints([0] * rows), ints([0] * rows))
        assert torch.equal(back[:, 1, 0, 0].float(), expect[:, 0])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("q_size,k_size,v_size,spread", [(1e-30, 1.0, 1.0, 0), (1e30, 1e-25, 1.0, 0), (1.0, 40.0, 1e-30, 0), (1.0, 1.0, 1e30, 0),
                                                         (1.0, 0.0, 1.0, 0), (30.0, 30.0, 1.0, 8), (1.0, 1.0, 1.0, 20)])
def test_decode_of_far_sizes(ops, dtype, head_dim, q_size, k_size, v_size, spread):
    """Queries, keys and values far from one; scores hundreds apart, in rising and falling order; values' scales that differ
    from position to position by up to 2^spread. Weights below 2^-30 of the largest weight times scale are dropped."""
    lengths, page = [777, 300], 16
    pages, table = spread_tables(lengths, page, 8)
    pool = random_pool(ops, "fp8", pages, 2, page, head_dim, 3)
    gen = torch.Generator(device="cuda").manual_seed(3)
    pool.scales[:, 0] *= k_size
    pool.scales[:, 1] *= v_size
    pool.scales[:, 1] *= torch.pow(2.0, (spread * torch.rand(pool.scales[:, 1].shape, generator=gen, device="cuda")).round())
    for r, n in enumerate(lengths):       # keys that grow along the first context and shrink along the second
        at = torch.arange(n)
        grow = (at + 1.0) / n if r == 0 else 1.0 - at / n
        pool.scales[table[r].cpu().long()[at // page].cuda(), 0, :, (at % page).cuda()] *= grow[:, None].cuda()
    q = (q_size * torch.randn((2, 6, head_dim), generator=gen, device="cuda")).to(dtype)
    out, positions = torch.zeros_like(q), ints([n - 1 for n in lengths])
    ops.paged_attention_decode(q, pool, out, table, ints([0, 1]), ints([0, 1]), positions, 0.2, 777)
    ops.check_status("cuda")
    exact, bound = exact_decode(q, pool, table, [(0, 0), (1, 1)], positions, 0.2)
    keys = pool.codes.float().abs().amax() * pool.scales[:, 0].nan_to_num().amax()
    size = float(q.float().abs().amax() * keys * head_dim * 0.2)      # of a score, at most
    largest = bound.amax(-1, keepdim=True)
    per_weight = (HALF[BF16] if dtype == BF16 else 0.0) + max(size, 30) * 8 * 2.0 ** -24
    limit = per_weight * bound + HALF[dtype] * exact.abs() * 1.01 + 2.0 ** -30 * 777 * largest
    assert ((out.double() - exact).abs() <= limit).all()


@gpu
@pytest.mark.parametrize("offset", [1, 8])
def test_operands_that_do_not_lie_on_16_bytes(ops, offset):
    """Slices of larger tensors, which the vector forms do not take."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    aligned = random_pool(ops, "fp8", 9, 2, 16, 64, 1)
    room = torch.zeros(aligned.codes.numel() + 16, dtype=torch.uint8, device="cuda")
    codes = room[offset:offset + aligned.codes.numel()].view(torch.float8_e4m3fn).view(aligned.shape)
    codes.view(torch.uint8).copy_(aligned.codes.view(torch.uint8))
    pool = ops.QuantizedPool(codes, aligned.scales.clone())
    table = ints([[3, 1, 7, 5, 0, 2, 8, 6, 4]])
    k = torch.randn((3, 2 * 64 + 1), generator=gen, device="cuda").to(BF16)[:, 1:]
    for p in (aligned, pool):
        ops.write_cache(k, k, p, ints([3 * 16, 3 * 16 + 1, 7 * 16 + 4]), ints([0, 1, 36]))
    assert torch.equal(pool.codes.view(torch.uint8), aligned.codes.view(torch.uint8)) and torch.equal(pool.scales, aligned.scales)
    backs = [torch.zeros(pool.shape, dtype=BF16, device="cuda") for _ in range(2)]
    for p, back in zip((aligned, pool), backs):
        ops.read_cache(p, back, table, ints([0]), ints([100]), ints([100]))
    assert torch.equal(*backs)
    wide = torch.randn(1 * 4 * 64 + 8, generator=gen, device="cuda").to(BF16)
    positions = ints([100])
    for p, q in ((pool, wide[:256].view(1, 4, 64)), (aligned, wide[1:257].view(1, 4, 64))):
        out = torch.zeros(1, 4, 64, dtype=BF16, device="cuda")
        ops.paged_attention_decode(q, p, out, table, ints([0]), ints([0]), positions, 0.125, 101)
        close(out, *exact_decode(q, p, table, [(0, 0)], positions, 0.125), BF16)
    ops.check_status("cuda")


@gpu
def test_pools_of_more_than_31_bits_of_bytes(ops):
    """Rows whose byte offsets need 32 bits and more: written, read back, attended to."""
    pages, kv_heads, page, head_dim = 70_000, 8, 16, 128
    codes = torch.zeros((pages, 2, kv_heads, page, head_dim), dtype=torch.int8, device="cuda")      # 2.3 GB
    pool = ops.QuantizedPool(codes, torch.zeros(codes.shape[:4], device="cuda"))
    assert codes.numel() > 1 << 31
    held = [69_999, 69_000, 3, 66_123]
    gen = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn((60, kv_heads * head_dim), generator=gen, device="cuda").to(BF16) for _ in range(2))
    ops.write_cache(k, v, pool, ints([held[t // 16] * 16 + t % 16 for t in range(60)]), ints(range(60)))
    table = ints([held])
    q = torch.randn((1, 16, head_dim), generator=gen, device="cuda").to(BF16)
    out = torch.zeros_like(q)
    ops.paged_attention_decode(q, pool, out, table, ints([0]), ints([0]), ints([59]), 0.1, 60)
    small = ops.QuantizedPool(codes[held].contiguous(), pool.scales[held].contiguous())      # the same rows in a pool of four pages
    order = ints([[0, 1, 2, 3]])
    close(out, *exact_decode(q, small, order, [(0, 0)], ints([59]), 0.1), BF16)
    back = torch.zeros(codes.shape, dtype=BF16, device="cuda")
    ops.read_cache(pool, back, table, ints([0]), ints([59]), ints([59]))
    expect = torch.zeros(small.shape, dtype=BF16, device="cuda")
    ops.read_cache(small, expect, order, ints([0]), ints([59]), ints([59]))
    assert torch.equal(back[held], expect) and back.count_nonzero() == expect.count_nonzero()
    ops.check_status("cuda")
    del back, codes, pool
    torch.cuda.empty_cache()


def _a_step(ops, kind, seed, tokens=5, heads=8, kv_heads=2, head_dim=128, page=16, width=40):
    """A decode step's buffers: projections, pool, tables, lists; the call that stores, attends and reads back."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pool = random_pool(ops, kind, tokens * width, kv_heads, page, head_dim, seed)
    order = torch.randperm(tokens * width, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    s = dict(pool=pool, table=order.view(tokens, width).cuda(), positions=ints([0] * tokens), slots=ints([0] * tokens),
             qkv=torch.zeros((tokens, (heads + 2 * kv_heads) * head_dim), dtype=BF16, device="cuda"),
             q=torch.zeros((tokens, heads, head_dim), dtype=BF16, device="cuda"),
             out=torch.zeros((tokens, heads, head_dim), dtype=BF16, device="cuda"),
             back=torch.zeros(pool.shape, dtype=BF16, device="cuda"), rows=ints(range(tokens)))
    angle = torch.rand((page * width, head_dim // 2), generator=gen, device="cuda")
    s["cos"], s["sin"] = angle.cos(), angle.sin()

    def feed(turn):
        """The next step's numbers, into the same buffers."""
        g = torch.Generator(device="cuda").manual_seed(100 * seed + turn)
        s["qkv"].copy_(torch.randn(s["qkv"].shape, generator=g, device="cuda"))
        at = torch.randint(0, page * width, (tokens,), generator=g, device="cuda")
        s["positions"].copy_(at)
        s["slots"].copy_(s["table"].long().gather(1, (at // page)[:, None])[:, 0] * page + at % page)

    def call():
        hq, hk = heads * head_dim, kv_heads * head_dim
        ops.qk_norm_rope_cache(s["qkv"][:, :hq], s["qkv"][:, hq:hq + hk], s["qkv"][:, hq + hk:], s["q"], pool, s["slots"], s["positions"],
                               None, None, s["cos"], s["sin"], 0.0)
        ops.paged_attention_decode(s["q"], pool, s["out"], s["table"], s["rows"], s["rows"], s["positions"], 0.09, page * width, settled=True)
        ops.read_cache(pool, s["back"], s["table"], s["rows"], s["positions"], s["positions"])

    def result():
        return [t.clone() for t in (s["q"], s["out"], s["back"], pool.codes.view(torch.uint8), pool.scales)]
    return feed, call, result


@gpu
@pytest.mark.parametrize("chained", [False, True])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_captured_steps_replay(ops, kind, chained):
    """Two captured graphs of two steps of their own, replayed in turn with new numbers, with and without launches that
    overlap: bit for bit what the calls themselves give."""
    eager = [_a_step(ops, kind, seed) for seed in (1, 2)]
    captured = [_a_step(ops, kind, seed) for seed in (1, 2)]
    try:
        ops.set_chained_launches(chained)
        graphs = []
        for feed, call, _ in captured:
            feed(0)
            call()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call()
            graphs.append(graph)
        for feed, call, _ in eager:
            feed(0)
            call()
        for turn in range(1, 6):
            for one, other, graph in zip(eager, captured, graphs):
                for feed, _, _ in (one, other):
                    feed(turn)
                one[1]()
                graph.replay()
        torch.cuda.synchronize()
        for one, other in zip(eager, captured):
            for a, b in zip(one[2](), other[2]()):
                assert torch.equal(a, b)
        ops.check_status("cuda")
    finally:
        ops.set_chained_launches(False)


@gpu
def test_steps_on_two_streams_at_once(ops):
    alone = [_a_step(ops, "fp8", seed) for seed in (3, 4)]
    beside = [_a_step(ops, "fp8", seed) for seed in (3, 4)]
    streams = [torch.cuda.Stream() for _ in beside]
    for feed, call, _ in alone:
        for turn in range(20):
            feed(turn)
            call()
    torch.cuda.synchronize()
    for turn in range(20):
        for (feed, call, _), stream in zip(beside, streams):
            with torch.cuda.stream(stream):
                feed(turn)
                call()
    torch.cuda.synchronize()
    for one, other in zip(alone, beside):
        for a, b in zip(one[2](), other[2]()):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("head_dim,heads,kv_heads", [(128, 8, 2), (256, 4, 2), (48, 4, 2)])
def test_rows_written_right_ahead_are_seen(ops, head_dim, heads, kv_heads):
    """With overlapping launches on, a write of whole contexts directly ahead of the attention: without ``settled`` it waits
    for all of it."""
    page, length, rows = 16, 1500, 6
    pages, table = spread_tables([length] * rows, page, 2)
    gen = torch.Generator(device="cuda").manual_seed(2)
    at = torch.arange(length).repeat(rows)
    slots = (table.cpu().long()[torch.arange(rows).repeat_interleave(length), at // page] * page + at % page).to(torch.int32).cuda()
    q = torch.randn((rows, heads, head_dim), generator=gen, device="cuda").to(BF16)
    positions = ints([length - 1] * rows)
    try:
        ops.set_chained_launches(True)
        for turn in range(4):
            pool = ops.QuantizedPool.zeros(pages, kv_heads, page, head_dim)
            k, v = (torch.randn((rows * length, kv_heads * head_dim), generator=gen, device="cuda").to(BF16) for _ in range(2))
            out = torch.zeros_like(q)
            torch.cuda.synchronize()
            ops.write_cache(k, v, pool, slots, at.to(torch.int32).cuda())
            ops.paged_attention_decode(q, pool, out, table, ints(range(rows)), ints(range(rows)), positions, 0.1, length)
            close(out, *exact_decode(q, pool, table, [(r, r) for r in range(rows)], positions, 0.1), BF16)
    finally:
        ops.set_chained_launches(False)
    ops.check_status("cuda")


@gpu
def test_calls_of_nothing(ops):
    pool = random_pool(ops, "fp8", 2, 2, 16, 64, 0)
    none, q = ints([]), torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    assert ops.paged_attention_decode(q, pool, q, ints([[0, 1]]), none, none, none, 0.1, 20) is q
    before = pool.scales.clone()
    empty = torch.zeros(0, 128, dtype=BF16, device="cuda")
    ops.write_cache(empty, empty, pool, none, none)
    out = torch.ones(pool.shape, device="cuda")
    ops.read_cache(pool, out, ints([[0, 1]]), none, none, none)
    ops.read_cache(pool, out, ints([[0, 1]]), ints([0]), ints([0]), ints([-1]))
    assert out.eq(1).all() and torch.equal(pool.scales, before)
    ops.check_status("cuda")


@gpu
@pytest.mark.parametrize("head_dim", [128, 40])
def test_reaches_beyond_31_bits_limit_nothing(ops, head_dim):
    """Windows, chunks and kept positions arrive whole: none becomes a small one by losing its upper half."""
    pool = random_pool(ops, "fp8", 20, 2, 16, head_dim, 3)
    table, lists = ints([list(range(20))]), (ints([0]), ints([0]), ints([299]))
    q = torch.randn((1, 4, head_dim), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(BF16)
    plain, back = torch.zeros_like(q), torch.zeros(pool.shape, dtype=BF16, device="cuda")
    ops.paged_attention_decode(q, pool, plain, table, *lists, 0.1, 300)
    ops.read_cache(pool, back, table, ints([0]), ints([299]), ints([299]))
    for options in (dict(window=2 ** 32 + 5), dict(chunk=2 ** 32 + 7), dict(window=2 ** 31), dict(window=2 ** 31 - 1),
                    dict(window=3, keep=2 ** 32 + 1), dict(chunk=16, keep=2 ** 31 - 1)):
        out, read = torch.zeros_like(q), torch.zeros_like(back)
        ops.paged_attention_decode(q, pool, out, table, *lists, 0.1, 300, **options)
        ops.read_cache(pool, read, table, ints([0]), ints([299]), ints([299]), **options)
        assert torch.equal(read, back), options
        # cuts of the sum differ: two results that are each within a rounding and the halves' 2^-10 of the exact one
        assert (out.float() - plain.float()).abs().max() <= 2.0 ** -7 * plain.float().abs().max() + 2.0 ** -9 * 4, options
    ops.check_status("cuda")


@gpu
def test_pools_of_heads_without_values_are_refused(ops):
    pool = ops.QuantizedPool(torch.zeros((2, 2, 1, 4, 0), dtype=torch.int8, device="cuda"), torch.zeros((2, 2, 1, 4), device="cuda"))
    k = torch.zeros((1, 0), dtype=BF16, device="cuda")
    with pytest.raises(ops.KernelError, match="between 1 and 512"):
        ops.write_cache(k, k, pool, ints([0]), ints([0]))


@gpu
@pytest.mark.parametrize("head_dim,heads,kv_heads,page", [(128, 8, 2, 16), (64, 7, 1, 8), (256, 4, 2, 32), (40, 4, 2, 4), (128, 4, 2, 3)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["fp8", None])
@pytest.mark.parametrize("longest", [70, 5000])
def test_a_padding_rows_request_is_not_looked_at(ops, kind, dtype, head_dim, heads, kv_heads, page, longest):
    """Padding rows whose request lies outside the block tables, over codes and over a cache in the compute type: bit for
    bit what padding rows of request 0 give."""
    if kind is None and not ops.decode_attention_supported(head_dim, heads, kv_heads, dtype):
        pytest.skip("the split-key kernel does not take this layout")
    lengths = [longest, 3]
    pages, table = spread_tables(lengths, page, 1)
    pool = random_pool(ops, "fp8", pages, kv_heads, page, head_dim, 2)
    if kind is None:
        pool = values_of(pool).to(dtype)
    q = torch.randn((4, heads, head_dim), generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(dtype)
    positions = ints([2, 0, longest - 1, 0])
    outs = []
    for filler in ([0, 0, 0], [-1, 2 ** 30, -2 ** 31], [2 ** 31 - 1, 2, -5]):
        out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
        ops.paged_attention_decode(q, pool, out, table, ints([-1, 2, -7, 0, -2 ** 31]), ints([filler[0], 0, filler[1], 1, filler[2]]),
                                   positions, 0.1, longest)
        outs.append(out)
    ops.check_status("cuda")
    assert outs[0][[1, 3]].eq(5.0).all() and not outs[0][[0, 2]].eq(5.0).all()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def close_as_halves(out, exact, bound, dtype, keys):
    """What the tensor-core form owes: bfloat16 queries' weights are halves (2^-11 each; below 2^-14, with the largest at
    2^6 or above, 2^-31 of the largest), float32 queries' two halves (2^-22); the rest as in ``close``."""
    per_weight = (2.0 ** -11 if dtype == BF16 else 2.0 ** -22) + 30 * 8 * 2.0 ** -24
    least = keys * 2.0 ** -31 * bound.amax(-1, keepdim=True)
    off = (out.double() - exact).abs()
    limit = per_weight * bound + least + HALF[dtype] * exact.abs() * 1.01 + 1e-30
    assert (off <= limit).all(), f"{(off / limit).max().item():.2f} times the bound"


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim,heads,kv_heads,page", [(64, 7, 1, 8), (128, 8, 2, 16), (256, 4, 2, 32)])
@pytest.mark.parametrize("options", [dict(), dict(window=900), dict(window=200, keep=300), dict(chunk=512)],
                         ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()) or "all")
def test_settled_positions_and_a_row_written_right_ahead(ops, kind, dtype, head_dim, heads, kv_heads, page, options):
    """A step as an engine makes it, with overlapping launches on: contexts written earlier, a copy, the tokens' own rows,
    and the attention, told that the contexts are settled. Against the definition, not against another run."""
    lengths = [1500, 1, 129, 700, 2048, 33]
    rows = len(lengths)
    pages, table = spread_tables(lengths, page, 2)
    gen = torch.Generator(device="cuda").manual_seed(2)
    at = torch.cat([torch.arange(n) for n in lengths])
    request = torch.cat([torch.full((n,), r) for r, n in enumerate(lengths)])
    slots = table.cpu().long()[request, at // page] * page + at % page
    own = at == torch.tensor(lengths)[request] - 1
    q = torch.randn((rows, heads, head_dim), generator=gen, device="cuda").to(dtype)
    positions, lists = ints([n - 1 for n in lengths]), ints(range(rows))
    host, older, newer = positions.cpu().pin_memory(), (~own).cuda(), own.cuda()
    slots_of = [slots[m].to(torch.int32).cuda() for m in (~own, own)]
    try:
        ops.set_chained_launches(True)
        for turn in range(3):
            pool = random_pool(ops, kind, pages, kv_heads, page, head_dim, 50 + turn)      # earlier owners' rows
            k, v = (torch.randn((len(at), kv_heads * head_dim), generator=gen, device="cuda").to(dtype) for _ in range(2))
            out = torch.zeros_like(q)
            parts = [(k[m], v[m]) for m in (older, newer)]
            wheres = [at[m].to(torch.int32).cuda() for m in (~own, own)]
            torch.cuda.synchronize()
            ops.write_cache(*parts[0], pool, slots_of[0], wheres[0])
            positions.copy_(host, non_blocking=True)       # a step's integers
            ops.write_cache(*parts[1], pool, slots_of[1], wheres[1])
            ops.paged_attention_decode(q, pool, out, table, lists, lists, positions, 0.1, max(lengths), settled=True, **options)
            ops.check_status("cuda")
            close_as_halves(out, *exact_decode(q, pool, table, [(r, r) for r in range(rows)], positions, 0.1, **options), dtype, max(lengths))
    finally:
        ops.set_chained_launches(False)


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("head_dim,heads,kv_heads,page", [(64, 14, 2, 32), (128, 16, 2, 16), (256, 5, 1, 8)])
@pytest.mark.parametrize("longest", [40, 900, 6000])
def test_weights_are_halves(ops, kind, head_dim, heads, kv_heads, page, longest):
    """bfloat16 outputs to within the eleven bits that weights are held in."""
    lengths = [longest, longest // 3 + 1, 1]
    pages, table = spread_tables(lengths, page, 4)
    pool = random_pool(ops, kind, pages, kv_heads, page, head_dim, 8)
    q = (1.5 * torch.randn((3, heads, head_dim), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")).to(BF16)
    positions, lists, out = ints([n - 1 for n in lengths]), ints(range(3)), torch.zeros_like(q)
    scale = 1.0 / math.sqrt(head_dim)
    ops.paged_attention_decode(q, pool, out, table, lists, lists, positions, scale, longest)
    ops.check_status("cuda")
    close_as_halves(out, *exact_decode(q, pool, table, [(r, r) for r in range(3)], positions, scale), BF16, longest)


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("padding,longest", [(1, 100), (3, 9000), (40, 9000)])
def test_attention_of_padding_alone_keeps_the_order_of_launches(ops, kind, padding, longest):
    """Overlapping launches: a write of whole contexts, an attention whose rows are all padding, and pages read back, which
    wait for the write although the attention between had nothing to do."""
    page, length, rows, kv_heads, head_dim = 16, 2000, 6, 4, 128
    pages, table = spread_tables([length] * rows, page, 2)
    gen = torch.Generator(device="cuda").manual_seed(4)
    at = torch.arange(length).repeat(rows)
    slots = (table.cpu().long()[torch.arange(rows).repeat_interleave(length), at // page] * page + at % page).to(torch.int32).cuda()
    at = at.to(torch.int32).cuda()
    q, out = (torch.zeros((padding, 8, head_dim), dtype=BF16, device="cuda") for _ in range(2))
    none, lists, last = ints([-1] * padding), ints(range(rows)), ints([length - 1] * rows)
    zeros, first = ints([0] * padding), ints([0] * rows)
    try:
        ops.set_chained_launches(True)
        for turn in range(6):
            pool = ops.QuantizedPool.zeros(pages, kv_heads, page, head_dim, codes=kind)
            k, v = (torch.randn((rows * length, kv_heads * head_dim), generator=gen, device="cuda").to(BF16) for _ in range(2))
            back = torch.zeros(pool.shape, dtype=F32, device="cuda")
            torch.cuda.synchronize()
            ops.write_cache(k, v, pool, slots, at)
            ops.paged_attention_decode(q, pool, out, table, none, zeros, zeros, 0.1, longest, settled=True)
            ops.read_cache(pool, back, table, lists, first, last)
            ops.check_status("cuda")
            assert torch.equal(back, values_of(pool).float()) and out.eq(0).all()
    finally:
        ops.set_chained_launches(False)


@gpu
@pytest.mark.parametrize("head_dim,offset", [(64, 0), (40, 0), (64, 1)])
@pytest.mark.parametrize("last", [8, 11, 4000, 2 ** 31 - 1])
@pytest.mark.parametrize("options", [dict(), dict(window=3), dict(keep=2, window=1)], ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()) or "all")
def test_positions_beyond_the_table_are_reported(ops, head_dim, offset, last, options):
    """By either kernel that reads pages back; what the table has of them is read, nothing else is written."""
    made = random_pool(ops, "fp8", 5, 2, 4, head_dim, 1)
    room = torch.zeros(made.codes.numel() + 16, dtype=torch.uint8, device="cuda")
    codes = room[offset:offset + made.codes.numel()].view(torch.float8_e4m3fn).view(made.shape)
    codes.view(torch.uint8).copy_(made.codes.view(torch.uint8))
    pool, table = ops.QuantizedPool(codes, made.scales), ints([[1, 3]])
    zero, far = ints([0]), ints([last])
    expect = torch.full(pool.shape, 7.0, device="cuda")
    expect[[1, 3]] = values_of(pool)[[1, 3]].float()
    out = torch.full(pool.shape, 7.0, device="cuda")
    ops.read_cache(pool, out, table, zero, zero, far, **options)
    with pytest.raises(ops.KernelError, match="block-table"):
        ops.check_status("cuda")
    assert torch.equal(out, expect)
    for tables, end in ((table, 7), (torch.empty((1, 0), dtype=torch.int32, device="cuda"), -1)):
        ops.read_cache(pool, out, tables, zero, zero, ints([end]), **options)
        ops.check_status("cuda")
    assert torch.equal(out, expect)
    ops.read_cache(pool, out, torch.empty((1, 0), dtype=torch.int32, device="cuda"), zero, zero, zero, **options)
    with pytest.raises(ops.KernelError, match="block-table"):
        ops.check_status("cuda")
    assert torch.equal(out, expect)


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim", [64, 128, 256, 40])
@pytest.mark.parametrize("signs", ["all", "keys", "mixed"])
def test_scales_of_either_sign(ops, kind, dtype, head_dim, signs):
    """A row stands for code * scale whatever the scale's sign: pools that a caller's own program made."""
    lengths = [700, 40]
    pages, table = spread_tables(lengths, 16, 1)
    pool = random_pool(ops, kind, pages, 2, 16, head_dim, 2)
    if signs == "mixed":
        pool.scales.mul_(torch.where(torch.rand(pool.scales.shape, generator=torch.Generator().manual_seed(3)) > 0.5, 1.0, -1.0).cuda())
    else:
        pool.scales[:, :1 if signs == "keys" else 2].neg_()
    q = torch.randn((2, 4, head_dim), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    out, positions, lists = torch.zeros_like(q), ints([n - 1 for n in lengths]), ints([0, 1])
    ops.paged_attention_decode(q, pool, out, table, lists, lists, positions, 0.1, 700)
    ops.check_status("cuda")
    exact, bound = exact_decode(q, pool, table, [(0, 0), (1, 1)], positions, 0.1)
    close_as_halves(out, exact, bound, dtype, 700)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim", [64, 128, 256, 40])
@pytest.mark.parametrize("size", [1e-32, 1e-34, 1e-36])
@pytest.mark.parametrize("where", ["all", "later", "earlier"])
def test_values_near_the_least_of_float32(ops, dtype, head_dim, size, where):
    """Values of such a size throughout, and beside ordinary ones that come ahead of them or behind."""
    lengths = [1500, 300]
    pages, table = spread_tables(lengths, 16, 1)
    pool = random_pool(ops, "fp8", pages, 2, 16, head_dim, 2)
    for r, n in enumerate(lengths):
        held = [int(p) for p in table[r, :-(-n // 16)]]
        small = held if where == "all" else held[len(held) // 2:] if where == "later" else held[:len(held) // 2]
        pool.scales[small, 1] *= size
    q = torch.randn((2, 4, head_dim), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    out, positions, lists = torch.zeros_like(q), ints([n - 1 for n in lengths]), ints([0, 1])
    ops.paged_attention_decode(q, pool, out, table, lists, lists, positions, 0.1, 1500)
    ops.check_status("cuda")
    exact, bound = exact_decode(q, pool, table, [(0, 0), (1, 1)], positions, 0.1)
    # p_j scale_j and, times 2^125, its halves end at 2^-150 each: so much a key, times a code, over a sum of one or more
    ends, off = 1500 * 448 * 2.0 ** -149, (out.double() - exact).abs()
    # times 2^100, so that sizes count as in other tests
    close_as_halves(torch.where(off <= ends, exact, out.double()) * 2.0 ** 100, exact * 2.0 ** 100, bound * 2.0 ** 100, dtype, 1500)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_dim", [64, 128, 256, 40])
@pytest.mark.parametrize("size", [1e32, 1e35, 3e37])
def test_queries_near_the_largest_of_float32(ops, dtype, head_dim, size):
    """Queries whose products with the codes pass float32's range while the scores do not, and the other way about."""
    lengths = [700, 40]
    pages, table = spread_tables(lengths, 16, 1)
    plain = random_pool(ops, "fp8", pages, 2, 16, head_dim, 2)
    q = torch.randn((2, 4, head_dim), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").clamp(-4, 4)
    positions, lists = ints([n - 1 for n in lengths]), ints([0, 1])
    for up in (size, 1.0 / size):
        pool = ops.QuantizedPool(plain.codes, plain.scales.clone())
        pool.scales[:, 0] /= up
        large, out = (q * up).to(dtype), torch.zeros(q.shape, dtype=dtype, device="cuda")
        ops.paged_attention_decode(large, pool, out, table, lists, lists, positions, 0.1, 700)
        ops.check_status("cuda")
        exact, bound = exact_decode(large, pool, table, [(0, 0), (1, 1)], positions, 0.1)
        close_as_halves(out, exact, bound, dtype, 700)


@gpu
@pytest.mark.parametrize("kind", ["fp8", None])
@pytest.mark.parametrize("head_dim,page,width", [(128, 16, 40), (64, 8, 3), (128, 16, 0), (256, 16, 5)])
def test_padding_alone_over_tables_without_rows(ops, kind, head_dim, page, width):
    pool = random_pool(ops, "fp8", 4, 2, page, head_dim, 1)
    dtype = BF16 if kind or head_dim < 256 else F32
    if kind is None:
        if not ops.decode_attention_supported(head_dim, 4, 2, dtype):
            pytest.skip("the split-key kernel does not take this layout")
        pool = values_of(pool).to(dtype)
    q = torch.zeros((2, 4, head_dim), dtype=dtype, device="cuda")
    out = torch.full_like(q, 3.0)
    table = torch.empty((0, width), dtype=torch.int32, device="cuda")
    for longest in (60, 6000):
        ops.paged_attention_decode(q, pool, out, table, ints([-1, -1, -3]), ints([-1, 7, 2 ** 31 - 1]), ints([0, 0]), 0.1, longest)
    ops.check_status("cuda")
    assert out.eq(3.0).all()
