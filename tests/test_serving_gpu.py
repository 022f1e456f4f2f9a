"""The serving-step operators on an MI355X against plain 64-bit forms.

Tolerances are bounds by arithmetic, computed beside each result: half a step
of the output's type, eps(t) / 2 relative; fp32 sums of n terms, n 2^-24 of the
sum of magnitudes; weights of the attention in fp16, 2^-11 of theirs.
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF16, FP16, FP32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
INF, NAN = math.inf, math.nan
E32 = 2.0**-24  # half a step of fp32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.fixture(scope="module")
def serving():
    from gpud_amd.diag import serving as s

    return s


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, want, bound):
    """Elementwise |got - want| <= bound, equal where `want` is not finite."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    off = (got - want).abs()[fine] - (bound.expand_as(want)[fine] if isinstance(bound, torch.Tensor) else bound)
    assert not off.numel() or float(off.max()) <= 0, f"beyond the bound by {float(off.max()):.3g}"


# ---------------------------------------------------------------------------
# w4_matmul
# ---------------------------------------------------------------------------


def w4_case(serving, m, n, k, group, zeros, dtype, seed=0, spread=1.0):
    g = gen(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda")
    groups = -(-k // group)
    scales = (torch.rand(n, groups, generator=g, device="cuda") * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 16, (n, groups), generator=g, device="cuda") if zeros else None
    x = (torch.randn(m, k, generator=g, device="cuda") * spread).to(dtype)
    packed = serving.pack_w4(codes, scales, z, group_size=group)
    column = torch.arange(k, device="cuda") // group
    zz = z.double()[:, column] if zeros else torch.full((n, k), 8.0, dtype=torch.float64, device="cuda")
    s = scales.double()[:, column]
    w = (codes.double() - zz) * s
    want = x.double() @ w.t()
    # every term of a group's fp32 sum is of x with 16 + q and with 16 + z, 2 group
    # terms; the groups' sums and the waves' are further terms
    size = x.double().abs() @ ((codes.double() + 32 + zz) * s).t()
    bound = half_step(dtype) * want.abs() + (2 * group + groups + 16) * E32 * size
    bound += (half_step(dtype) * bound) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
    return x, packed, want, bound


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize(
    "m,n,k,group",
    [
        (1, 1, 1, 32), (1, 16, 128, 128), (2, 17, 127, 32), (3, 33, 129, 64), (16, 100, 1000, 128), (17, 64, 520, 64),
        (31, 40, 264, 32), (33, 50, 2048, 128), (64, 90, 1024, 32), (65, 30, 640, 64), (130, 20, 384, 128), (1, 4100, 2056, 128),
        (16, 2070, 300, 64), (48, 1030, 4096, 32), (5, 7, 9000, 128),
    ],
)
def test_w4_matmul(serving, m, n, k, group, zeros, dtype):
    x, (codes, scales, z), want, bound = w4_case(serving, m, n, k, group, zeros, dtype, seed=m * n + k)
    got = serving.w4_matmul(x, codes, scales, z, out_features=n, group_size=group)
    assert got.dtype == dtype and got.shape == (m, n)
    close(got, want, bound)
    again = serving.w4_matmul(x, codes, scales, z, out_features=n, group_size=group)
    assert torch.equal(got, again)


@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("n", (40, 8200, 16400))
@pytest.mark.parametrize("m", (18, 50, 70))
def test_w4_matmul_of_many_tokens(serving, m, n, group, zeros):
    # 1, 2 and 4 tiles of rows a workgroup; the columns end inside a group, and
    # there are fewer blocks of them than workgroups that begin apart
    k, dtype = 1500, BF16 if m == 50 else FP16
    x, (codes, scales, z), want, bound = w4_case(serving, m, n, k, group, zeros, dtype, seed=m + n + group)
    got = serving.w4_matmul(x, codes, scales, z, out_features=n, group_size=group)
    close(got, want, bound)
    assert torch.equal(got, serving.w4_matmul(x, codes, scales, z, out_features=n, group_size=group))


@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("tiles", (257, 520, 521, 770, 1030, 1300, 1788, 1794, 2100))
@pytest.mark.parametrize("m", (2, 16, 29, 61))
def test_w4_matmul_of_any_number_of_rows(serving, m, tiles, group, zeros):
    # from 1 to 8 tiles of rows a workgroup, the last of them not there or not whole
    n, k, dtype = tiles * 16 - 5, 1100, FP16 if m == 16 else BF16
    x, (codes, scales, z), want, bound = w4_case(serving, m, n, k, group, zeros, dtype, seed=m + n + group)
    close(serving.w4_matmul(x, codes, scales, z, out_features=n, group_size=group), want, bound)


def test_w4_matmul_of_the_most_columns(serving):
    # as many scales and zero points as the LDS holds
    n, k = 16 * 600, serving.MAX_COLUMNS
    for m in (1, 16, 40):
        x, (codes, scales, z), want, bound = w4_case(serving, m, n, k, 32, True, BF16, seed=m)
        close(serving.w4_matmul(x, codes, scales, z, out_features=n, group_size=32), want, bound)
        del want, bound


def test_w4_matmul_strides_offsets_and_out(serving):
    m, n, k = 5, 40, 256
    x, (codes, scales, z), want, bound = w4_case(serving, m, n, k, 64, True, BF16)
    wide = torch.full((m, k + 24), NAN, dtype=BF16, device="cuda")
    for at in (0, 8, 3):  # aligned rows, and rows that 16-byte loads do not fit
        wide[:, at:at + k] = x
        close(serving.w4_matmul(wide[:, at:at + k], codes, scales, z, out_features=n, group_size=64), want, bound)
    odd = torch.full((m, k + 13), NAN, dtype=BF16, device="cuda")
    odd[:, 1:1 + k] = x
    close(serving.w4_matmul(odd[:, 1:1 + k], codes, scales, z, out_features=n, group_size=64), want, bound)
    close(serving.w4_matmul(x.t().contiguous().t(), codes, scales, z, out_features=n, group_size=64), want, bound)
    out = torch.full((m, n + 9), 7.0, dtype=BF16, device="cuda")
    r = serving.w4_matmul(x, codes, scales, z, out_features=n, group_size=64, out=out[:, 3:3 + n])
    close(r, want, bound)
    assert bool((out[:, :3] == 7).all()) and bool((out[:, 3 + n:] == 7).all())
    assert serving.w4_matmul(x[:0], codes, scales, z, out_features=n, group_size=64).shape == (0, n)


def test_w4_matmul_large_values_and_zero_rows(serving):
    x, (codes, scales, z), want, bound = w4_case(serving, 4, 64, 512, 128, True, BF16, spread=1e30)
    close(serving.w4_matmul(x, codes, scales, z, out_features=64), want, bound)
    x[1] = 0
    got = serving.w4_matmul(x, codes, scales, z, out_features=64)
    assert bool((got[1] == 0).all())
    # a NaN stays in its own row
    x[2, 5] = NAN
    got = serving.w4_matmul(x, codes, scales, z, out_features=64)
    assert bool(torch.isnan(got[2]).all()) and not bool(torch.isnan(got[[0, 1, 3]]).any())


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 16, 20, 50])
def test_w4_matmul_of_the_largest_values(serving, m, group, zeros):
    """Values just under 2^115 of one sign: the sums of a group stay within fp32."""
    n, k = 40, 500
    x = torch.full((m, k), 2.0**115, dtype=torch.float64, device="cuda").to(BF16)
    x = (x.double() * (1 - 2.0**-8)).to(BF16)
    x[m // 2] *= -1
    codes = torch.randint(0, 16, (n, k), generator=gen(m), device="cuda")
    codes[1] = torch.arange(k, device="cuda") % 2 * 2 + 7
    codes[2], codes[3] = 0, 15
    groups = -(-k // group)
    scales = torch.full((n, groups), 2.0**-6, dtype=BF16, device="cuda")
    z = torch.full((n, groups), 8, device="cuda")
    if zeros:
        z[4], z[5] = 0, 15
    packed = serving.pack_w4(codes, scales, z if zeros else None, group_size=group)
    zz = z.double()[:, torch.arange(k, device="cuda") // group]
    want = x.double() @ ((codes.double() - zz) / 64).t()
    size = x.double().abs() @ ((codes.double() + 32 + zz) / 64).t()
    bound = half_step(BF16) * want.abs() + (2 * group + groups + 16) * E32 * size
    got = serving.w4_matmul(x, *packed, out_features=n, group_size=group)
    close(got, want, bound * (1 + half_step(BF16)))


# ---------------------------------------------------------------------------
# cache
# ---------------------------------------------------------------------------


class Cache:
    """A cache with a shuffled table, filled by the operator, and its plain mirror."""

    def __init__(self, serving, lens, heads, dim, page, seed=0, spare=2, blocks=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        blocks = blocks or max(need + [1])
        total = sum(need) + spare
        order = torch.randperm(total, generator=g).tolist()
        table = torch.full((len(lens), blocks), -7, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                table[b, i] = order.pop()
        self.table, self.page, self.heads, self.dim = table.cuda(), page, heads, dim
        self.tensors = serving.new_cache(total, heads, dim, page)
        junk = torch.Generator(device="cuda").manual_seed(seed + 1)
        for t in self.tensors[:2]:  # what earlier owners left
            t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=junk, device="cuda", dtype=torch.uint8))

    def values(self, b, length):
        """Keys and values of a sequence in 64 bits, [heads, length, dim] each."""
        k, v, ks, vs = self.tensors
        ids = self.table[b, : -(-length // self.page)].long()
        kk = k.view(torch.uint8)[ids].view(F8).double() * ks[ids].double()[..., None, None]
        vv = v.view(torch.uint8)[ids].view(F8).double() * vs[ids].double()[..., None, None]
        kk = kk.transpose(0, 1).reshape(self.heads, -1, self.dim)[:, :length]
        vv = vv.permute(1, 0, 3, 2).reshape(self.heads, -1, self.dim)[:, :length]
        return kk, vv


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts_of(counts):
    s = [0]
    for n in counts:
        s.append(s[-1] + n)
    return s


def filled(serving, lens, heads, dim, page, dtype=BF16, seed=0, blocks=None):
    c = Cache(serving, lens, heads, dim, page, seed, blocks=blocks)
    g = gen(seed + 2)
    k, v = (torch.randn(sum(lens), heads, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    serving.cache_append(k, v, *c.tensors, c.table, ints(lens), ints(starts_of(lens)))
    return c, k, v


def plain_append(cache, scales, x, table, lens, starts, page, values):
    """The append's definition, page by page, in 64 bits up to the last rounding."""
    for b, length in enumerate(lens):
        count = starts[b + 1] - starts[b]
        first = length - count
        for block in range(max(first, 0) // page, (length + page - 1) // page):
            lo, hi = max(first, block * page, 0), min(length, block * page + page)
            p = int(table[b, block])
            if lo >= hi or not 0 <= p < cache.shape[0]:
                continue
            body = cache.view(torch.uint8)[p].view(F8).double()
            body = body.transpose(1, 2) if values else body  # [head, token, dim]
            new = x[starts[b] + lo - first:starts[b] + hi - first].double().transpose(0, 1)
            amax = torch.where(torch.isfinite(new), new.abs(), 0.0).amax((1, 2))
            e = torch.where(amax > 0, torch.ceil(torch.log2((amax / 448).clamp_min(2.0**-200))), -64.0).clamp_min(-64)
            e = torch.where(amax > 448 * torch.exp2(e), e + 1, torch.where((amax <= 224 * torch.exp2(e)) & (e > -64), e - 1, e))
            old = torch.log2(scales[p].double())
            if lo > block * page:
                e = torch.maximum(e, old)
                body = (body * torch.exp2(old - e)[:, None, None]).float().to(F8).double()
            body = body.clone()
            body[:, lo - block * page:hi - block * page] = (new * torch.exp2(-e)[:, None, None]).clamp(-448, 448).float().to(F8).double()
            scales[p] = torch.exp2(e).float()
            body = body.transpose(1, 2) if values else body
            cache[p] = body.float().to(F8)


def same_codes(a, b):
    """Codes that stand for the same values; NaN's two codes are one."""
    a, b = a.view(torch.uint8), b.view(torch.uint8)
    nan = (a & 127) == 127
    return torch.equal(nan, (b & 127) == 127) and torch.equal(a[~nan], b[~nan])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,dim,page", [(1, 16, 16), (2, 64, 16), (3, 80, 32), (2, 128, 64), (1, 256, 128), (1, 16, 512), (2, 64, 256)])
def test_cache_append_in_steps(serving, heads, dim, page, dtype):
    """Prompts, chunks that end inside pages, and single tokens, each of another size."""
    g = gen(dim + page)
    final = [1, page, page + 1, 5 * page - 3, 2, 0]
    cache = Cache(serving, [n + 40 for n in final], heads, dim, page, seed=page)
    mirror = [t.clone() for t in cache.tensors]
    table = cache.table.cpu()
    lens = [0] * len(final)
    for step in range(7):
        counts = final if step == 0 else [(step * (b + 2)) % 7 for b in range(len(final))] if step < 4 else [1] * len(final)
        counts = [min(n, t + 40 - cur) for n, t, cur in zip(counts, final, lens)]
        lens = [a + b for a, b in zip(lens, counts)]
        starts = starts_of(counts)
        both = torch.randn(starts[-1], 2, heads, dim, generator=g, device="cuda") * 2.0 ** (2 * step - 4)
        both = both.to(dtype)
        k, v = both[:, 0], both[:, 1]
        single = all(n == 1 for n in counts)
        serving.cache_append(k, v, *cache.tensors, cache.table, ints(lens), None if single else ints(starts))
        plain_append(mirror[0], mirror[2], k, table, lens, starts, page, False)
        plain_append(mirror[1], mirror[3], v, table, lens, starts, page, True)
        assert torch.equal(cache.tensors[2], mirror[2]) and torch.equal(cache.tensors[3], mirror[3])
        assert same_codes(cache.tensors[0], mirror[0])
        assert same_codes(cache.tensors[1], mirror[1])


def test_cache_append_extremes(serving):
    """Zeros, the smallest and largest values, infinities and NaN."""
    heads, dim, page = 1, 16, 16
    big = torch.finfo(BF16).max
    for rows in ([0.0] * 16, [INF, 1.0] + [0.0] * 14, [-INF, NAN] + [2.0] * 14, [big, -big, 1.0, 1e-38] * 4, [1e-38] * 16, [3.0, NAN] * 8):
        cache = Cache(serving, [3], heads, dim, page)
        mirror = [t.clone() for t in cache.tensors]
        k = torch.tensor(rows, dtype=BF16, device="cuda").expand(3, 1, 16).contiguous()
        serving.cache_append(k, -k, *cache.tensors, cache.table, ints([3]), ints([0, 3]))
        plain_append(mirror[0], mirror[2], k, cache.table.cpu(), [3], [0, 3], page, False)
        plain_append(mirror[1], mirror[3], -k, cache.table.cpu(), [3], [0, 3], page, True)
        assert torch.equal(cache.tensors[2], mirror[2]) and torch.equal(cache.tensors[3], mirror[3])
        assert same_codes(cache.tensors[0], mirror[0]) and same_codes(cache.tensors[1], mirror[1])


def test_cache_append_leaves_out_bad_pages_and_other_rows(serving):
    heads, dim, page = 2, 32, 16
    cache = Cache(serving, [40, 40, 40], heads, dim, page, spare=1)
    table = cache.table.clone()
    table[0, 1] = -1
    table[1, 0] = cache.tensors[0].shape[0]
    table[2, 2] = 2**31 - 1
    before = [t.clone() for t in cache.tensors]
    k = torch.randn(125, heads, dim, device="cuda").to(BF16)  # 5 rows behind the last sequence
    serving.cache_append(k, k, *cache.tensors, table, ints([40, 40, 40]), ints([0, 40, 80, 120]))
    touched = {int(table[b, i]) for b in range(3) for i in range(3) if 0 <= int(table[b, i]) < cache.tensors[0].shape[0]}
    for p in range(cache.tensors[0].shape[0]):
        same = all(torch.equal(t[p].view(torch.uint8), u[p].view(torch.uint8)) for t, u in zip(cache.tensors, before))
        assert same == (p not in touched)
    # longer than the table's row, and empty
    serving.cache_append(k, k, *cache.tensors, table, ints([48 + 40, 0, -5]), ints([0, 40, 80, 120]))


def test_cache_append_of_sequences_longer_than_their_table(serving):
    """Their tokens up to its end are written, and nothing of empty ones or of negative lengths."""
    heads, dim, page = 2, 32, 16
    cache = Cache(serving, [40, 40, 40], heads, dim, page, spare=1)
    mirror = [t.clone() for t in cache.tensors]
    k = torch.randn(125, heads, dim, generator=gen(4), device="cuda").to(BF16)
    lens, starts = [48 + 17, 0, -5], [0, 40, 80, 120]
    serving.cache_append(k, -k, *cache.tensors, cache.table, ints(lens), ints(starts))
    for i, x in ((0, k), (1, -k)):
        plain_append(mirror[i], mirror[i + 2], x, cache.table.cpu()[:1], [48], [0, 48 - (65 - 40)], page, bool(i))
        assert torch.equal(cache.tensors[i + 2], mirror[i + 2]) and same_codes(cache.tensors[i], mirror[i])


# ---------------------------------------------------------------------------
# cache_attention
# ---------------------------------------------------------------------------


def check_attention(cache, q, lens, starts, got, scale=None, window=None, skip=()):
    out, lse = got
    heads, dim = cache.heads, cache.dim
    group = q.shape[1] // heads
    scale = dim**-0.5 if scale is None else scale
    for b, length in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        if lo == hi or b in skip:
            continue
        qq = q[lo:hi].double().view(-1, heads, group, dim).permute(1, 2, 0, 3)
        pos = torch.arange(length - (hi - lo), length, device="cuda")
        if length == 0:
            close(out[lo:hi], torch.zeros_like(out[lo:hi]), 0.0)
            assert bool((lse[lo:hi] == -INF).all())
            continue
        k, v = cache.values(b, length)
        j = torch.arange(length, device="cuda")
        hidden = j > pos[:, None]
        if window:
            hidden |= j <= pos[:, None] - window
        score = (qq @ k[:, None].transpose(2, 3)) * scale
        size = (qq.abs() @ k[:, None].abs().transpose(2, 3)) * abs(scale)
        score = score.masked_fill(hidden, -INF)
        total = torch.logsumexp(score, -1, keepdim=True)
        p = torch.exp(score - total).masked_fill(hidden, 0.0)
        p = torch.where(torch.isnan(p), 0.0, p)
        clean = torch.where(hidden.all(0)[:, None], 0.0, v)
        want = p @ clean[:, None]
        # of a score: its fp32 sum and the steps to the power of two; then the sum of weights
        shift = float((size.masked_fill(hidden, 0).amax() * (dim + 8) + score.masked_fill(hidden, 0).abs().amax() * 4) * E32)
        rel = math.expm1(shift) + 2.0**-21 + (length + 8) * E32
        mass = p @ clean[:, None].abs()
        # fp16 weights: 2^-11 of each, and 2^-25 of the largest one for those under its range
        top = p.amax(-1, keepdim=True) * clean.abs().amax((-2, -1))[:, None, None, None]
        bound = mass * (2.0**-11 + 2 * rel) + top * length * 2.0**-25 * 2
        bound = bound + half_step(out.dtype) * (want.abs() + bound) + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
        o = out[lo:hi].view(-1, heads, group, dim).permute(1, 2, 0, 3)
        close(o, want, bound)
        s = lse[lo:hi].view(-1, heads, group).permute(1, 2, 0)
        t = total.squeeze(-1)
        close(s, t, rel + torch.where(torch.isfinite(t), t.abs(), 0.0) * 4 * E32)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize(
    "heads,group,dim,page",
    [(1, 1, 16, 16), (2, 8, 64, 16), (2, 4, 128, 64), (1, 16, 128, 32), (3, 5, 80, 16), (1, 40, 64, 128), (2, 2, 256, 64), (1, 3, 208, 32), (8, 4, 96, 16)],
)
def test_attention_single_tokens(serving, heads, group, dim, page, dtype):
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 300, 1111, 2]
    cache, _, _ = filled(serving, lens, heads, dim, page, dtype, seed=dim + group)
    q = torch.randn(len(lens), heads * group, dim, generator=gen(3), device="cuda").to(dtype)
    for longest in (None, 1, 5000):
        got = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), max_seq_len=longest)
        check_attention(cache, q, lens, list(range(len(lens) + 1)), got)
    again = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), max_seq_len=5000)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("window", [None, 1, 50, 64, 400])
@pytest.mark.parametrize("heads,group,dim,page", [(2, 4, 128, 64), (1, 1, 64, 16), (2, 8, 64, 32), (1, 7, 128, 16), (1, 32, 256, 16), (2, 3, 208, 16), (1, 16, 80, 64), (3, 1, 48, 128)])
def test_attention_chunks(serving, heads, group, dim, page, window, dtype):
    lens = [700, 1, 33, 0, 64, 500, 129]
    counts = [5, 1, 33, 0, 20, 150, 1]
    cache, _, _ = filled(serving, lens, heads, dim, page, dtype, seed=dim + group)
    starts = starts_of(counts)
    q = torch.randn(starts[-1], heads * group, dim, generator=gen(4), device="cuda").to(dtype)
    got = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), ints(starts), window=window)
    check_attention(cache, q, lens, starts, got, window=window)


def test_attention_long_prompt_and_scale(serving):
    lens = counts = [1500]
    cache, _, _ = filled(serving, lens, 2, 128, 64)
    q = torch.randn(1500, 8, 128, generator=gen(4), device="cuda").to(BF16)
    got = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), ints([0, 1500]), scale=0.3)
    check_attention(cache, q, lens, starts_of(counts), got, scale=0.3)


def test_attention_scales_of_every_size(serving):
    """Pages whose scales differ by many powers of two, in keys and in values."""
    page, lens = 16, [200, 77]
    cache = Cache(serving, lens, 2, 64, page, seed=9)
    g = gen(10)
    k, v = (torch.randn(277, 2, 64, generator=g, device="cuda") for _ in range(2))
    at = torch.cat([torch.arange(n, device="cuda") for n in lens])
    k *= torch.exp2(((at // page) % 5).float() - 3)[:, None, None]
    v *= torch.exp2(((at // page) * 7 % 23).float() - 12)[:, None, None]
    serving.cache_append(k.to(BF16), v.to(BF16), *cache.tensors, cache.table, ints(lens), ints(starts_of(lens)))
    q = torch.randn(2, 8, 64, generator=g, device="cuda").to(BF16)
    check_attention(cache, q, lens, [0, 1, 2], serving.cache_attention(q, *cache.tensors, cache.table, ints(lens)))


def test_attention_strides_and_rows_behind_the_last(serving):
    lens, counts = [100, 40], [3, 2]
    cache, _, _ = filled(serving, lens, 2, 64, 16)
    starts = starts_of(counts)
    fused = torch.randn(9, 8 + 4, 64, generator=gen(5), device="cuda").to(BF16)
    q = fused[:, :8]  # 4 rows behind the last sequence
    out, lse = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), ints(starts))
    check_attention(cache, q[:5], lens, starts, (out, lse))
    assert bool((out[5:] == 0).all()) and bool((lse[5:] == -INF).all())
    mine = torch.full((9, 8, 64), 5.0, dtype=BF16, device="cuda")
    out2, _ = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), ints(starts), out=mine)
    assert out2 is mine and torch.equal(mine[:5], out[:5]) and bool((mine[5:] == 5).all())
    odd = torch.zeros(9 * 8 * 64 + 3, dtype=BF16, device="cuda")[3:].view(9, 8, 64)  # not aligned to 16 bytes
    odd.copy_(q)
    assert torch.equal(serving.cache_attention(odd, *cache.tensors, cache.table, ints(lens), ints(starts))[0], out)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(serving.cache_attention(turned, *cache.tensors, cache.table, ints(lens), ints(starts))[0], out)
    table = torch.cat([cache.table, cache.table], 1)[:, : cache.table.shape[1]]
    assert torch.equal(serving.cache_attention(q, *cache.tensors, table, ints(lens), ints(starts))[0], out)


@pytest.mark.parametrize("window", [None, 30])
def test_attention_masked_nan_reaches_only_rows_that_see_it(serving, window):
    """A NaN among cached values or keys shows in the rows that see it alone."""
    lens, counts = [150], [90]
    for which in ("k", "v"):
        cache = Cache(serving, lens, 1, 64, 16)
        k, v = (torch.randn(150, 1, 64, generator=gen(i), device="cuda").to(BF16) for i in (1, 2))
        (k if which == "k" else v)[100, 0, 7] = NAN
        serving.cache_append(k, v, *cache.tensors, cache.table, ints(lens), ints([0, 150]))
        q = torch.randn(90, 4, 64, generator=gen(3), device="cuda").to(BF16)
        out, lse = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), ints([0, 90]), window=window)
        pos = torch.arange(60, 150, device="cuda")
        sees = (pos >= 100) & ((pos < 130) if window else True)
        bad = torch.isnan(out)
        assert not bool(bad[~sees].any())
        if which == "v":
            assert bool(bad[sees][..., 7].all()) and not bool(bad[..., [i for i in range(64) if i != 7]].any())
            assert not bool(torch.isnan(lse).any())
        else:
            assert bool(bad[sees].all()) and torch.equal(torch.isnan(lse), sees[:, None].expand_as(lse))


def test_attention_bad_pages_and_lengths(serving):
    lens = [100, 100, 100, 100]
    cache, _, _ = filled(serving, lens, 2, 64, 16)
    table = cache.table.clone()
    table[1, 3] = -1
    table[2, 6] = cache.tensors[0].shape[0]
    q = torch.randn(4, 4, 64, generator=gen(1), device="cuda").to(BF16)
    said = [100, 100, 100, 7 * 16 + 1]  # the last is longer than its row of the table
    out, lse = serving.cache_attention(q, *cache.tensors, table, ints(said))
    check_attention(cache, q[:1], lens[:1], [0, 1], (out[:1], lse[:1]))
    assert bool(torch.isnan(out[1:]).all()) and bool(torch.isnan(lse[1:]).all())
    # pages behind a sequence's end are not looked at; a negative length is an empty sequence
    table = cache.table.clone()
    table[0, 1:] = 2**31 - 1
    out, lse = serving.cache_attention(q, *cache.tensors, table, ints([16, 5, -3, 100]))
    assert not bool(torch.isnan(out).any()) and bool((out[2] == 0).all()) and bool((lse[2] == -INF).all())


@pytest.mark.parametrize("count", [1, 5, 40, 100])
def test_attention_longer_than_its_table_is_nan(serving, count):
    """Every row of such a sequence, also with no table at all; its neighbours are not touched."""
    cache, _, _ = filled(serving, [120, 120], 2, 64, 16)
    q = torch.randn(2 * count, 8, 64, generator=gen(1), device="cuda").to(BF16)
    starts = [0, count, 2 * count]
    out, lse = serving.cache_attention(q, *cache.tensors, cache.table, ints([8 * 16 + 1, 120]), ints(starts))
    assert bool(torch.isnan(out[:count]).all()) and bool(torch.isnan(lse[:count]).all())
    check_attention(cache, q, [120, 120], starts, (out, lse), skip=(0,))
    for blocks in (0, 1):
        out, lse = serving.cache_attention(q, *cache.tensors, cache.table[:, :blocks], ints([120, 0]), ints(starts))
        assert bool(torch.isnan(out[:count]).all()) and bool(torch.isnan(lse[:count]).all())
        assert bool((out[count:] == 0).all()) and bool((lse[count:] == -INF).all())


@pytest.mark.parametrize("window", [None, 70])
def test_attention_mixed_batches_of_long_chunks(serving, window):
    """Sequences of many rows and of few take passes of their own; rows behind them too."""
    lens, counts = [600, 90, 1, 0, 333, 70, 2000], [300, 1, 1, 0, 7, 70, 130]
    for dim, group in ((128, 4), (64, 8), (208, 3)):
        cache, _, _ = filled(serving, lens, 2, dim, 32, seed=dim)
        starts = starts_of(counts)
        q = torch.randn(starts[-1] + 9, 2 * group, dim, generator=gen(2), device="cuda").to(BF16)
        for longest in (None, 1):
            got = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), ints(starts), window=window, max_seq_len=longest)
            check_attention(cache, q, lens, starts, got, window=window)
            assert bool((got[0][starts[-1]:] == 0).all()) and bool((got[1][starts[-1]:] == -INF).all())
        mine = torch.full_like(q, 3.0)
        serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), ints(starts), window=window, out=mine)
        check_attention(cache, q, lens, starts, (mine, got[1]), window=window)
        assert bool((mine[starts[-1]:] == 3).all())


def test_attention_masked_nan_in_long_chunks(serving):
    lens, counts = [400], [200]
    cache = Cache(serving, lens, 1, 128, 64)
    k, v = (torch.randn(400, 1, 128, generator=gen(i), device="cuda").to(BF16) for i in (1, 2))
    v[300, 0, 77] = NAN
    serving.cache_append(k, v, *cache.tensors, cache.table, ints(lens), ints([0, 400]))
    q = torch.randn(200, 4, 128, generator=gen(3), device="cuda").to(BF16)
    for window in (None, 30):
        out, lse = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), ints([0, 200]), window=window)
        pos = torch.arange(200, 400, device="cuda")
        sees = (pos >= 300) & ((pos < 330) if window else True)
        bad = torch.isnan(out)
        assert torch.equal(bad[..., 77], sees[:, None].expand(-1, 4)) and int(bad.sum()) == int(sees.sum()) * 4
        assert not bool(torch.isnan(lse).any())


def test_attention_offsets_past_32_bits(serving):
    """Pages whose bytes lie beyond 2^31 and 2^32."""
    heads, dim, page = 8, 128, 64
    pages = 2**32 // (heads * dim * page) + 40
    cache = Cache.__new__(Cache)
    cache.heads, cache.dim, cache.page = heads, dim, page
    cache.tensors = serving.new_cache(pages, heads, dim, page)
    cache.table = torch.tensor([[pages - 1, 5, pages // 2 + 3], [0, pages - 2, 1]], dtype=torch.int32, device="cuda")
    lens = [150, 190]
    k, v = (torch.randn(340, heads, dim, generator=gen(i), device="cuda").to(BF16) for i in (1, 2))
    serving.cache_append(k, v, *cache.tensors, cache.table, ints(lens), ints(starts_of(lens)))
    kk, _ = cache.values(0, 150)
    amax = k[:150].double().abs().amax()
    assert float((kk - k[:150].double().transpose(0, 1)).abs().max()) <= float(amax) * 2.0**-4
    q = torch.randn(2, 32, dim, generator=gen(3), device="cuda").to(BF16)
    check_attention(cache, q, lens, [0, 1, 2], serving.cache_attention(q, *cache.tensors, cache.table, ints(lens)))


def test_attention_empty_batches(serving):
    cache, _, _ = filled(serving, [20], 2, 64, 16)
    none = torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    out, lse = serving.cache_attention(none, *cache.tensors, cache.table[:0], ints([]))
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    some = torch.randn(3, 4, 64, device="cuda").to(BF16)
    out, lse = serving.cache_attention(some, *cache.tensors, cache.table[:0], ints([]), ints([0]))
    assert bool((out == 0).all()) and bool((lse == -INF).all())
    out, lse = serving.cache_attention(some, *cache.tensors, cache.table, ints([0]), ints([0, 3]))
    assert bool((out == 0).all()) and bool((lse == -INF).all())


@pytest.mark.parametrize("which", ["decode", "chunk"])
@pytest.mark.parametrize("dim,group", [(80, 4), (208, 2), (48, 1), (16, 16), (112, 20)])
def test_attention_masked_nan_keys_of_any_dimension(serving, dim, group, which):
    """A NaN key behind the window stays behind it, wherever it lies in its tile."""
    window, length, count = 21, 120, 1 if which == "decode" else 5
    batch = 40
    lens, counts = [length + b % 3 for b in range(batch)], [count] * batch
    cache = Cache(serving, lens, 2, dim, 16)
    starts = starts_of(lens)
    k, v = (torch.randn(sum(lens), 2, dim, generator=gen(i), device="cuda").to(BF16) for i in (1, 2))
    seen = []
    for b, n in enumerate(lens):
        first = n - count - window  # the last position that no row sees
        at = first - b // 2 if b < 36 else first + 1 + b % 4
        k[starts[b] + at, :, b % 16] = NAN
        if b >= 36:
            seen.append(b)
    serving.cache_append(k, v, *cache.tensors, cache.table, ints(lens), ints(starts))
    rows = starts_of(counts)
    q = torch.randn(rows[-1], 2 * group, dim, generator=gen(3), device="cuda").to(BF16)
    out, lse = serving.cache_attention(
        q, *cache.tensors, cache.table, ints(lens), None if count == 1 else ints(rows), window=window
    )
    check_attention(cache, q, lens, rows, (out, lse), window=window, skip=seen)
    for b in seen:
        for i in range(count):
            pos = lens[b] - count + i
            sees = lens[b] - count - window + 1 + b % 4 > pos - window
            assert bool(torch.isnan(out[rows[b] + i]).all()) == sees and bool(torch.isnan(lse[rows[b] + i]).all()) == sees


@pytest.mark.parametrize("counts", [[3, 2], [3, 200], [100], [1, 1]])
def test_attention_lse_of_rows_behind_the_last(serving, counts):
    """With `out` given they keep what it held, and their lse is -inf as without it."""
    lens = [n + 30 for n in counts]
    for dim in (64, 208):
        cache, _, _ = filled(serving, lens, 2, dim, 16)
        starts = starts_of(counts)
        q = torch.randn(starts[-1] + 70, 8, dim, generator=gen(5), device="cuda").to(BF16)
        mine = torch.full_like(q, 5.0)
        for _ in range(3):
            before = torch.full((q.shape[0], 8), 7.0, device="cuda")  # what the next tensor of this size is made of
            del before
            _, lse = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), ints(starts), out=mine)
            check_attention(cache, q, lens, starts, (mine, lse))
            assert bool((mine[starts[-1]:] == 5).all()) and bool((lse[starts[-1]:] == -INF).all())


@pytest.mark.parametrize("value", [0.0, -1.0, INF, NAN])
@pytest.mark.parametrize("dim,count", [(64, 1), (64, 5), (128, 100), (80, 3), (80, 90), (208, 2)])
def test_attention_scales_of_pages_that_no_row_sees(serving, dim, count, value):
    """Pages behind the window and behind the last token hold whatever a program left there."""
    window, lens, counts = 10, [190, 60 + count], [count, count]
    cache, _, _ = filled(serving, lens, 2, dim, 16, blocks=13)
    table = cache.table
    spare = set(range(cache.tensors[0].shape[0])) - set(table.flatten().tolist())
    table[table < 0] = spare.pop()  # a page that nothing was written to
    _, _, ks, vs = cache.tensors
    kept = [t.clone() for t in (ks, vs)]
    for b, n in enumerate(lens):
        for block in range(13):
            if block * 16 + 15 <= n - count - window or block * 16 >= n:
                ks[int(table[b, block])] = vs[int(table[b, block])] = value
    starts = starts_of(counts)
    q = torch.randn(starts[-1], 8, dim, generator=gen(3), device="cuda").to(BF16)
    got = serving.cache_attention(q, *cache.tensors, table, ints(lens), None if count == 1 else ints(starts), window=window)
    ks.copy_(kept[0]), vs.copy_(kept[1])
    check_attention(cache, q, lens, starts, got, window=window)


@pytest.mark.parametrize("rows", [1, 100])
def test_attention_of_many_small_weights_beside_a_large_one(serving, rows):
    """One token with half of the weight, and 1.6 million others that share the rest."""
    length, dim, page = 1605000, 64, 4096
    cache = Cache(serving, [length], 1, dim, page, spare=0)
    k, v = torch.zeros(length, 1, dim, dtype=FP16, device="cuda"), torch.ones(length, 1, dim, dtype=FP16, device="cuda")
    k[0, 0, 0] = 14.0
    v[0] = -0.25
    serving.cache_append(k, v, *cache.tensors, cache.table, ints([length]), ints([0, length]))
    q = torch.zeros(rows, 1, dim, dtype=FP16, device="cuda")
    q[:, :, 0] = math.log(length) / 14
    for longest in (1, None):
        out, lse = serving.cache_attention(
            q, *cache.tensors, cache.table, ints([length]), ints([0, rows]), scale=1.0, max_seq_len=longest
        )
        pos = torch.arange(length - rows, length, device="cuda", dtype=torch.float64)[:, None]
        sink = torch.exp(q[:, 0, :1].double() * 14)
        want = (pos - 0.25 * sink) / (pos + sink)
        # fp16 weights, 2^-11 of each; fp32 sums, of a product 2 terms and of the weights
        # one a tile of 64 tokens; the score's fp32 sum and power
        mass = (pos + 0.25 * sink) / (pos + sink)
        rel = (length / 64 + 64 + 14.3 * 2 * (dim + 8)) * E32
        bound = float((mass * (2.0**-11 + 2 * rel) + want.abs() * rel).max()) + half_step(FP16)
        print(float((out[:, 0].double() - want).abs().max()), bound)
        assert float((out[:, 0].double() - want).abs().max()) <= bound
        close(lse, torch.log(pos + sink), rel + 16 * 4 * E32)


def test_attention_at_the_limits_of_its_values(serving):
    lens, page = [70, 40], 16
    cache = Cache(serving, lens, 2, 64, page)
    g = gen(8)
    k, v = (torch.randn(110, 2, 64, generator=g, device="cuda") for _ in range(2))
    at = torch.cat([torch.arange(n, device="cuda") for n in lens])
    v *= torch.where(at // page % 2 == 0, 0.0, 3e12)[:, None, None]
    serving.cache_append(k.to(BF16), v.to(BF16), *cache.tensors, cache.table, ints(lens), ints(starts_of(lens)))
    largest = cache.tensors[3].amax()
    assert 2.0**-64 * 2.0**98 <= float(largest) <= 2.0**-64 * 2.0**100
    q = torch.randn(2, 8, 64, generator=g, device="cuda").to(BF16)
    check_attention(cache, q, lens, [0, 1, 2], serving.cache_attention(q, *cache.tensors, cache.table, ints(lens)))
    q = torch.full_like(q, 2.0**109)  # scores of one sign and the largest size
    key = torch.full((110, 2, 64), 1.75 * 2.0**-64 * 2.0**8, dtype=BF16, device="cuda")
    serving.cache_append(key, v.to(BF16), *cache.tensors, cache.table, ints(lens), ints(starts_of(lens)))
    assert bool((cache.tensors[2][cache.table[0].long()] == 2.0**-64).all())
    got = serving.cache_attention(q, *cache.tensors, cache.table, ints(lens), scale=2.0**-60)
    check_attention(cache, q, lens, [0, 1, 2], got, scale=2.0**-60)


# ---------------------------------------------------------------------------
# token_logprobs
# ---------------------------------------------------------------------------


def check_logprobs(r, x, t, top):
    y = x.double()
    vocab = y.shape[1]
    p = torch.log_softmax(y, -1)
    void = (y == -INF).all(1)
    p[void] = -INF
    inside = (t >= 0) & (t < vocab)
    tt = torch.where(inside, t, 0)
    want = p.gather(1, tt[:, None]).squeeze(1)
    want = torch.where(inside, want, torch.where(t < 0, 0.0, NAN))
    # a lane's 64 terms, the tree of lanes and spans, the exponential and logarithm;
    # x - m and the logarithm of the sum are at most |log p| + log V
    rel = (64 + 12 + vocab // 2048 // 64 + 12 + 16) * E32

    def bound_of(lp):
        return rel + (torch.where(torch.isfinite(lp), lp.abs(), 0.0) + math.log(vocab) + 8) * 4 * E32

    close(r.logprob, want, bound_of(want))
    bound = bound_of(torch.zeros((), dtype=torch.float64, device=y.device))
    q = torch.exp(p)
    ent = -(torch.where(q > 0, q * p, torch.zeros_like(p))).sum(1)
    ent = torch.where(torch.isnan(p).any(1), NAN, torch.where(void, 0.0, ent))
    close(r.entropy, ent, bound * (4 + 2 * math.log(vocab + 1)))
    above = (y > y.gather(1, tt[:, None])).sum(1)
    assert torch.equal(r.rank, torch.where(inside, above, -1))
    if not top:
        assert r.top_ids is None and r.top_logprobs is None
        return
    order = torch.where(torch.isnan(y), INF, y) + 0.0
    nan_first = torch.sort(torch.isnan(y).to(torch.uint8), dim=1, descending=True, stable=True)
    ids = torch.sort(order, dim=1, descending=True, stable=True).indices
    if bool(torch.isnan(y).any()):  # NaN before everything, then by value
        rank = torch.sort(order.gather(1, nan_first.indices), dim=1, descending=True, stable=True).indices
        ids = nan_first.indices.gather(1, rank)
    ids = ids[:, :top]
    assert torch.equal(r.top_ids, ids)
    close(r.top_logprobs, p.gather(1, ids), bound_of(p.gather(1, ids)))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize(
    "rows,vocab,top",
    [(1, 1, 1), (3, 2, 0), (2, 7, 7), (5, 64, 64), (4, 65, 20), (7, 1000, 5), (3, 4096, 64), (2, 4097, 1), (3, 8191, 50), (9, 32000, 20), (2, 130001, 64), (1, 300007, 10)],
)
def test_token_logprobs(serving, rows, vocab, top, dtype):
    g = gen(vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    r = serving.token_logprobs(x, t, top)
    check_logprobs(r, x, t, top)
    again = serving.token_logprobs(x, t, top)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(r, again))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("vocab", [130, 5000, 20011])
def test_token_logprobs_masks_ties_and_padding(serving, dtype, vocab):
    g = gen(vocab)
    x = torch.randn(12, vocab, generator=g, device="cuda").to(dtype)
    x[0] = -INF  # nothing allowed
    x[1] = 0.0  # all the same
    x[2] = torch.where(torch.arange(vocab, device="cuda") % 2 == 0, 0.0, -0.0).to(dtype)
    x[3] = torch.arange(vocab, device="cuda").to(dtype) / 64  # rising
    x[4] = -torch.arange(vocab, device="cuda").to(dtype) / 64  # falling
    x[5] = -INF
    x[5, vocab // 3] = 2.0  # one allowed
    x[6, torch.rand(vocab, generator=g, device="cuda") < 0.95] = -INF
    x[7] = torch.finfo(dtype).min
    x[8] = 100.0 * x[8]
    x[9, : vocab // 2] = -INF
    x[10] = torch.round(x[10])  # many ties
    t = torch.randint(0, vocab, (12,), generator=g, device="cuda")
    t[5] = vocab // 3
    t[9] = 1  # a token that is not allowed
    check_logprobs(serving.token_logprobs(x, t, 50), x, t, 50)
    t[1], t[2], t[3], t[6] = -1, -100, vocab, 2**40
    check_logprobs(serving.token_logprobs(x, t, 3), x, t, 3)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_token_logprobs_nan_and_infinity(serving, dtype):
    x = torch.randn(5, 9001, generator=gen(1), device="cuda").to(dtype)
    x[0, 77] = NAN
    x[1, 8000] = INF
    x[2, 3] = NAN
    x[2, 8999] = INF
    x[3] = NAN
    t = torch.tensor([5, 8000, 9, 0, 1], device="cuda")
    check_logprobs(serving.token_logprobs(x, t, 20), x, t, 20)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_token_logprobs_strides_and_offsets(serving, dtype):
    g = gen(2)
    wide = torch.full((6, 10000), NAN, dtype=dtype, device="cuda")
    for at in range(0, 9):
        v = 8300 + at
        wide.fill_(NAN)
        wide[:, at:at + v] = (torch.randn(6, v, generator=g, device="cuda") * 2).to(dtype)
        x = wide[:, at:at + v]
        t = torch.randint(0, v, (6,), generator=g, device="cuda")
        check_logprobs(serving.token_logprobs(x, t, 12), x, t, 12)
    x = wide[:, 8:8308].t().contiguous().t()
    t = torch.randint(0, 8300, (12,), generator=g, device="cuda")[::2]
    check_logprobs(serving.token_logprobs(x, t, 4), x, t, 4)
    same = wide[:1, 8:8308].expand(6, -1)
    check_logprobs(serving.token_logprobs(same, t, 4), same, t, 4)
    empty = serving.token_logprobs(x[:0], t[:0], 4)
    assert empty.logprob.shape == (0,) and empty.top_ids.shape == (0, 4)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("vocab,top", [(5, 5), (700, 64), (5000, 30), (20011, 60), (32761, 3)])
def test_token_logprobs_are_the_same_among_few_rows_and_many(serving, dtype, vocab, top):
    # few rows take one launch, many take two
    g = gen(vocab)
    x = torch.randn(257, vocab, generator=g, device="cuda").to(dtype)
    x[0] = -INF
    x[1] = 1.0
    x[2] = torch.arange(vocab, device="cuda").to(dtype)
    x[3] = torch.finfo(dtype).min
    x[4, vocab // 2:] = -INF
    x[5] = torch.round(x[5])
    x[6, vocab // 3] = NAN
    x[7, vocab // 3] = INF
    t = torch.randint(0, vocab, (257,), generator=g, device="cuda")
    t[8], t[9] = -1, vocab
    many = serving.token_logprobs(x, t, top)
    for a, b in zip(many, serving.token_logprobs(x[:256], t[:256], top)):
        assert torch.equal(a[:256].nan_to_num(7e7), b.nan_to_num(7e7)) if a.is_floating_point() else torch.equal(a[:256], b)
    check_logprobs(serving.TokenLogprobs(*(v[8:] for v in many)), x[8:], t[8:], top)


@pytest.mark.parametrize("vocab", [65528, 65529, 65530, 65537])
def test_token_logprobs_at_the_most_spans_of_one_launch(serving, vocab):
    g = gen(vocab)
    wide = torch.randn(3, vocab + 9, generator=g, device="cuda").to(FP16)
    t = torch.randint(0, vocab, (3,), generator=g, device="cuda")
    for at in (0, 1, 7):
        x = wide[:, at:at + vocab]
        check_logprobs(serving.token_logprobs(x, t, 40), x, t, 40)


def test_token_logprobs_many_rows(serving):
    x = torch.randn(70000, 33, generator=gen(6), device="cuda").to(BF16)
    t = torch.randint(0, 33, (70000,), generator=gen(7), device="cuda")
    check_logprobs(serving.token_logprobs(x, t, 2), x, t, 2)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows", [30, 290])
def test_token_logprobs_of_large_magnitudes(serving, rows, dtype):
    """Finite masks over whole spans, and rows whose largest logit is far from 0; few rows and many."""
    g, vocab = gen(rows), 9001
    x = torch.randn(rows, vocab, generator=g, device="cuda")
    for i, mask in enumerate((-5e9, -1e10, -1e12, -1e20, -1e30)):
        x[4 * i] = mask  # nothing is allowed
        x[4 * i + 1, :4096] = mask  # a whole span
        x[4 * i + 2, 8192:] = mask  # the last one, which is not whole
        x[4 * i + 3] = mask
        x[4 * i + 3, 5000] = 1.0
    x[20, 77], x[21, 8900], x[22, 4096] = 1e10, 1e30, 9e36
    x[23] += 0.9e6
    x[24] += 1.1e6
    x[25] = x[25] * 10 - 3e7
    x[26] *= 1e10
    x[27] *= 1e30
    x[28] = x[28] * 1e36 - 9e36
    x = x.to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    t[3:20:4] = 5000
    t[20], t[21] = 77, 3
    check_logprobs(serving.token_logprobs(x, t, 20), x, t, 20)


# ---------------------------------------------------------------------------
# together, as a program uses them
# ---------------------------------------------------------------------------


class Step:
    """One layer and head of a model in low precision, and its decode step."""

    def __init__(self, serving, batch=6, width=256, heads=2, group=4, dim=64, vocab=5003, page=16):
        g = gen(77)
        self.s, self.dim, self.heads, self.q_heads = serving, dim, heads, heads * group
        qkv = (self.q_heads + 2 * heads) * dim

        def weights(n, k):
            codes = torch.randint(0, 16, (n, k), generator=g, device="cuda")
            scales = (torch.rand(n, -(-k // 64), generator=g, device="cuda") * 0.02 + 0.005).to(BF16)
            return (n,) + serving.pack_w4(codes, scales, group_size=64)

        self.qkv, self.o, self.head = weights(qkv, width), weights(width, self.q_heads * dim), weights(vocab, width)
        self.lens = [40, 3, 64, 100, 17, 0][:batch]
        self.cache = Cache(serving, [n + 10 for n in self.lens], heads, dim, page)
        self.x = torch.randn(batch, width, generator=g, device="cuda").to(BF16)
        self.targets = torch.randint(0, vocab, (batch,), generator=g, device="cuda")
        self.at = ints(self.lens)
        counts = self.lens
        k = torch.randn(sum(counts), heads, dim, generator=g, device="cuda").to(BF16)
        serving.cache_append(k, k * 0.5, *self.cache.tensors, self.cache.table, self.at, ints(starts_of(counts)))

    def product(self, x, w):
        return self.s.w4_matmul(x, w[1], w[2], w[3], out_features=w[0], group_size=64)

    def __call__(self):
        self.at += 1
        y = self.product(self.x, self.qkv).view(len(self.lens), -1, self.dim)
        q, k, v = y.split([self.q_heads, self.heads, self.heads], 1)
        self.s.cache_append(k, v, *self.cache.tensors, self.cache.table, self.at)
        o, _ = self.s.cache_attention(q, *self.cache.tensors, self.cache.table, self.at, max_seq_len=128)
        logits = self.product(self.product(o.flatten(1), self.o), self.head)
        return (q, k, v, o, logits) + tuple(self.s.token_logprobs(logits, self.targets, 5))


def test_step_matches_its_parts(serving):
    step = Step(serving)
    for n in range(1, 4):
        q, k, v, o, logits, *r = step()
        lens = [x + n for x in step.lens]
        alone = serving.cache_attention(q, *step.cache.tensors, step.cache.table, ints(lens), max_seq_len=128)
        check_attention(step.cache, q, lens, list(range(7)), alone)
        assert torch.equal(alone[0], o)
        for b, length in enumerate(lens):  # the step's own key is in the cache, within a rounding
            kk, _ = step.cache.values(b, length)
            page_max = kk.abs().amax()
            assert float((kk[:, -1] - k[b].double()).abs().max()) <= float(page_max) * 2.0**-4 + 2.0**-60
        from gpud_amd.diag.serving import TokenLogprobs

        check_logprobs(TokenLogprobs(*r), logits, step.targets, 5)


def test_step_in_two_graphs_and_on_another_stream(serving):
    """Captured twice and replayed among eager work, each replay equals the eager step."""
    eager = Step(serving)
    want = [[t.clone() for t in eager()] for _ in range(6)]
    one, two = Step(serving), Step(serving)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in (one, two):
            start = [t.clone() for t in s.cache.tensors]
            s()  # warm
            s.at -= 1
            for t, u in zip(s.cache.tensors, start):
                t.view(torch.uint8).copy_(u.view(torch.uint8)) if t.dtype == F8 else t.copy_(u)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for s in (one, two):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = s()
        graphs.append((graph, got))
    for n in range(6):
        for graph, got in graphs:
            graph.replay()
        scratch = torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")  # eager work between
        torch.cuda.synchronize()
        del scratch
        for graph, got in graphs:
            for a, b in zip(got, want[n]):
                assert torch.equal(a, b)
    third = Step(serving)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = third()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))


def test_tensors_without_memory_are_refused(serving):
    """Freed storages, in place of each tensor of each call."""

    def each(call, *tensors):
        call(*tensors)
        for i, t in enumerate(tensors):
            gone = torch.empty_like(t)
            gone.untyped_storage().resize_(0)
            with pytest.raises(ValueError, match="no memory"):
                call(*tensors[:i], gone, *tensors[i + 1:])

    x, (codes, scales, z), _, _ = w4_case(serving, 40, 48, 1100, 64, True, BF16)
    out = x.new_empty(40, 48)
    each(lambda x, c, s, z, o: serving.w4_matmul(x, c, s, z, out_features=48, group_size=64, out=o), x, codes, scales, z, out)
    cache, k, v = filled(serving, [40, 70], 2, 64, 16)
    lens, starts = ints([40, 70]), ints([0, 40, 110])
    each(serving.cache_append, k, v, *cache.tensors, cache.table, lens, starts)
    each(serving.cache_append, k[:2], v[:2], *cache.tensors, cache.table, lens)
    q = torch.randn(110, 4, 64, device="cuda").to(BF16)
    each(lambda *t: serving.cache_attention(*t[:-1], out=t[-1]), q, *cache.tensors, cache.table, lens, starts, q.clone())
    logits, targets = torch.randn(300, 100, device="cuda"), torch.zeros(300, dtype=torch.long, device="cuda")
    each(lambda x, t: serving.token_logprobs(x, t, 3), logits, targets)
    torch.cuda.synchronize()


def test_inference_without_gradients_and_with(serving):
    x, (codes, scales, z), want, bound = w4_case(serving, 2, 16, 128, 128, False, BF16)
    x.requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        serving.w4_matmul(x, codes, scales, out_features=16)
    with torch.no_grad():
        close(serving.w4_matmul(x, codes, scales, out_features=16), want, bound)


# ---------------------------------------------------------------------------
# the diagnostic
# ---------------------------------------------------------------------------


def test_serving_step_verifies_and_compares():
    from gpud_amd.diag import _serving

    for seed in (1, 2):
        res = _serving.serving_step(iters=3, seed=seed)
        assert res["verified"] and res["verify_failures"] == 0, res
        assert res["checked"] > 1_000_000 and res["gbps"] > 0
    wrong = _serving.serving_step(iters=1, oracle_offset=0.5)  # the oracle is off, on the host
    assert not wrong["verified"] and wrong["verify_failures"] > 100 and wrong["messages"]
    with pytest.raises(ValueError):
        _serving.serving_step(iters=0)


def test_serving_component_on_gpu():
    from gpud_amd.apiv1.types import HealthStateType
    from gpud_amd.bootstrap import build_core

    core = build_core(in_memory_db=True, kmsg_writable=False, record_reboot=False)
    try:
        comp = core.registry.get("accelerator-amd-diag-serving")
        assert comp is not None
        cr = comp.trigger_check()
        assert cr.health == HealthStateType.HEALTHY, f"{cr.reason} / {cr.error}"
        assert float(cr.extra_info["gpu0.step_gbps"]) > 0
    finally:
        core.close()
