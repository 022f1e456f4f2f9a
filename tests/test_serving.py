"""The serving-step operators on the host: layouts, work partition, refusals.

The partition of work (which workgroup has which rows, tokens and pages) is
plain arithmetic that the kernels share with host checks, so that lengths,
starts and page tables of every kind, broken ones too, are tried here.
"""

import random

import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("gpud_amd.diag._serving", reason="native extension not built")

from gpud_amd.diag import _serving, serving  # noqa: E402

BF16, FP16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


# -- layouts -----------------------------------------------------------------


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (16, 128, 128), (17, 129, 64), (40, 300, 32), (100, 513, 128)])
def test_pack_w4_keeps_every_code_in_its_documented_place(n, k, group):
    g = torch.Generator().manual_seed(n * k)
    codes = torch.randint(0, 16, (n, k), generator=g)
    groups = -(-k // group)
    scales = torch.rand(n, groups, generator=g).to(BF16)
    zeros = torch.randint(0, 16, (n, groups), generator=g)
    packed, s, z = serving.pack_w4(codes, scales, zeros, group_size=group)
    assert packed.shape == (-(-n // 16), -(-k // 128), 64, 16) and packed.is_contiguous()
    assert torch.equal(serving.unpack_w4(packed, n, k), codes.to(torch.uint8))
    rng = random.Random(k)
    for _ in range(200):
        row, col = rng.randrange(n), rng.randrange(k)
        b, c = divmod(col, 128)
        j, lanes, e = c // 32, c % 32 // 8, c % 8
        nibble = e // 2 + 4 * (e % 2)
        byte = int(packed[row // 16, b, 16 * lanes + row % 16, 4 * j + nibble // 2])
        assert byte >> 4 * (nibble % 2) & 15 == int(codes[row, col])
        assert s[row // 16, col // group, row % 16] == scales[row, col // group]
        assert z[row // 16, col // group, row % 16] == zeros[row, col // group]


def test_pack_w4_refuses_what_does_not_fit():
    codes, scales = torch.zeros(16, 128, dtype=torch.long), torch.ones(16, 1, dtype=BF16)
    for bad in (codes + 16, codes - 1):
        with pytest.raises(ValueError, match="0..15"):
            serving.pack_w4(bad, scales)
    with pytest.raises(ValueError, match="group_size"):
        serving.pack_w4(codes, scales, group_size=16)
    with pytest.raises(ValueError, match="scales"):
        serving.pack_w4(codes, scales, group_size=64)
    with pytest.raises(ValueError, match="zeros"):
        serving.pack_w4(codes, scales, torch.zeros(16, 2))
    with pytest.raises(ValueError, match="whole numbers"):
        serving.pack_w4(codes.float(), scales)
    with pytest.raises(ValueError, match="empty"):
        serving.pack_w4(codes[:0], scales[:0])


def test_cache_scale_is_the_smallest_power_of_two_that_fits():
    amax = torch.tensor([0.0, 1e-30, 1.0, 448.0, 448.1, 449.0, 3.5, 3.5001, 7.0, 1e30, 2.0**-64 * 448])
    got = serving.cache_scale(amax)
    assert torch.equal(torch.frexp(got).mantissa, torch.full_like(got, 0.5))
    assert bool((amax <= 448 * got).all())
    assert bool(((amax > 224 * got) | (got == 2.0**-64)).all())


# -- partition ---------------------------------------------------------------


def _random_batch(rng):
    batch = rng.choice([1, 2, 3, 7, 20])
    counts = [rng.choice([0, 1, 1, 2, 5, 33, 200]) for _ in range(batch)]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    lens = [max(0, n + rng.choice([-3, 0, 0, 1, 63, 64, 300, 900])) for n in counts]
    return starts, lens


@pytest.mark.parametrize("seed", range(40))
def test_attention_gives_each_row_its_tokens_once(seed):
    rng = random.Random(seed)
    starts, lens = _random_batch(rng)
    group, heads = rng.choice([1, 3, 4, 8, 16, 40]), 2
    tail = rng.choice([0, 1, 50])
    rows = starts[-1] + tail
    if not rows:
        return
    page, blocks, window = rng.choice([16, 64]), 80, rng.choice([0, 1, 64, 100])
    fill = rng.random() < 0.5
    got = _serving.attention_places(starts, lens, rows, heads, heads * group, page, blocks, window, rng.choice([1, 700, 5000]), fill)
    spans = {}
    for row, head, slot, split, lo, hi in got:
        spans.setdefault((row, head), []).append((split, lo, hi))
    want = rows if fill else starts[-1]
    assert set(spans) == {(r, h) for r in range(want) for h in range(group)}
    for b, length in enumerate(lens):
        count = starts[b + 1] - starts[b]
        for i in range(count):
            pos = length - count + i
            for h in range(group):
                parts = sorted(spans[starts[b] + i, h])
                assert [p[0] for p in parts] == list(range(len(parts)))
                for p, q in zip(parts, parts[1:]):
                    assert p[2] == q[1] and p[2] % 64 == 0
                lo = max(0, pos - window + 1) if window else 0
                assert parts[0][1] <= lo and parts[-1][2] > pos if pos >= 0 else True
                assert parts[-1][2] <= max(length, 0)


@pytest.mark.parametrize("seed", range(40))
def test_attention_of_any_dimension_gives_each_row_its_tokens_once(seed):
    """Wide heads have tiles of 16 rows and more of them a sequence; single tokens too."""
    rng = random.Random(seed)
    dim, heads = rng.choice([16, 64, 80, 128, 144, 208, 256]), rng.choice([1, 3])
    group = rng.choice([1, 3, 8, 16, 17, 32, 40, 64, 65, 130])
    starts, lens = _random_batch(rng)
    single = rng.random() < 0.3
    if single:
        starts = list(range(len(lens) + 1))
    tail = 0 if single else rng.choice([0, 7])
    rows = starts[-1] + tail
    if not rows:
        return
    window = rng.choice([0, 1, 64, 100])
    got = _serving.attention_places(
        [] if single else starts, lens, rows, heads, heads * group, 16, 80, window, rng.choice([1, 700, 5000]), True, dim
    )
    spans = {}
    for row, head, slot, split, lo, hi in got:
        spans.setdefault((row, head), []).append((split, lo, hi))
    assert set(spans) == {(r, h) for r in range(rows) for h in range(group)}
    for b, length in enumerate(lens):
        for i in range(starts[b], starts[b + 1]):
            pos = length - starts[b + 1] + i
            for h in range(group):
                parts = sorted(spans[i, h])
                assert [p[0] for p in parts] == list(range(len(parts)))
                assert all(p[2] == q[1] for p, q in zip(parts, parts[1:]))
                assert pos < 0 or parts[0][1] <= max(0, pos - window + 1 if window else 0) and parts[-1][2] > pos
                assert parts[-1][2] <= max(length, 0)


@pytest.mark.parametrize("seed", range(30))
def test_attention_survives_any_starts_and_lengths(seed):
    """Broken metadata may leave rows out; it never names a row that is not there."""
    rng = random.Random(seed)
    batch, rows = rng.choice([1, 4]), 50
    wild = lambda: rng.choice([-(2**31), -5, 0, 3, 49, 50, 51, 60, 10**6])  # noqa: E731
    starts = [wild() for _ in range(batch + 1)]
    lens = [rng.choice([-(2**31), -1, 0, 5, 64, 10**6, 2**31 - 1]) for _ in range(batch)]
    for row, head, slot, split, lo, hi in _serving.attention_places(starts, lens, rows, 2, 8, 16, 8, rng.choice([0, 5]), 100, True):
        assert 0 <= row < rows and 0 <= head < 4 and 0 <= lo and hi <= 128


@pytest.mark.parametrize("seed", range(40))
def test_append_gives_each_new_token_its_slot_once(seed):
    rng = random.Random(seed)
    starts, lens = _random_batch(rng)
    page, blocks = rng.choice([16, 64]), 80
    rows = starts[-1] + rng.choice([0, 9])
    batch = len(lens)
    table = list(range(batch * blocks))
    rng.shuffle(table)
    got = {}
    for slot, pid, lo, hi, src in _serving.append_places(starts, lens, table, rows, page, blocks, batch * blocks):
        assert 0 <= lo < hi <= page
        for i in range(lo, hi):
            assert (pid, i) not in got
            got[pid, i] = src + i - lo
    want = {}
    for b, length in enumerate(lens):
        count = starts[b + 1] - starts[b]
        for i in range(count):
            pos = length - count + i
            if pos >= 0:
                want[table[b * blocks + pos // page], pos % page] = starts[b] + i
    assert got == want


@pytest.mark.parametrize("seed", range(30))
def test_append_survives_any_metadata(seed):
    rng = random.Random(seed)
    batch, rows, blocks, page, pages = rng.choice([1, 4]), 50, 3, 16, 6
    starts = [rng.choice([-(2**31), -5, 0, 3, 49, 50, 51, 10**6]) for _ in range(batch + 1)]
    lens = [rng.choice([-(2**31), -1, 0, 5, 48, 49, 2**31 - 1]) for _ in range(batch)]
    table = [rng.choice([-1, 0, 5, 6, 2**31 - 1]) for _ in range(batch * blocks)]
    for slot, pid, lo, hi, src in _serving.append_places(starts, lens, table, rows, page, blocks, pages):
        assert 0 <= pid < pages and 0 <= lo < hi <= page and 0 <= src and src + hi - lo <= rows


# -- refusals ----------------------------------------------------------------


def w4_args(**change):
    a = dict(
        x=torch.zeros(3, 256, dtype=BF16), codes=torch.zeros(2, 2, 64, 16, dtype=torch.uint8),
        scales=torch.zeros(2, 2, 16, dtype=BF16), zeros=None, out_features=20, group_size=128,
    )
    a.update(change)
    return a


@pytest.mark.parametrize(
    "change,error,match",
    [
        (dict(), ValueError, "on a GPU"),
        (dict(x=[1.0]), TypeError, "tensor"),
        (dict(x=torch.zeros(3, 256)), TypeError, "float32"),
        (dict(x=torch.zeros(256, dtype=BF16)), ValueError, "2 dimensions"),
        (dict(x=torch.zeros(3, 0, dtype=BF16)), ValueError, "no product"),
        (dict(x=torch.zeros(3, 300, dtype=BF16)), ValueError, "codes has shape"),
        (dict(x=torch.zeros(1, 256, dtype=BF16).expand(65473, 256)), ValueError, "no product"),
        (dict(x=torch.zeros(1, 32769, dtype=BF16)), ValueError, "no product"),
        (dict(out_features=0), ValueError, "no product"),
        (dict(out_features=33), ValueError, "codes has shape"),
        (dict(group_size=100), ValueError, "group_size"),
        (dict(group_size=64), ValueError, "scales has shape"),
        (dict(scales=torch.zeros(2, 2, 16, dtype=FP16)), TypeError, "scales"),
        (dict(codes=torch.zeros(2, 2, 64, 32, dtype=torch.uint8)[..., ::2]), ValueError, "contiguous"),
        (dict(zeros=torch.zeros(2, 2, 16)), TypeError, "zeros"),
        (dict(zeros=torch.zeros(2, 1, 16, dtype=torch.uint8)), ValueError, "zeros has shape"),
        (dict(zeros=torch.zeros(65, dtype=torch.uint8)[1:].view(2, 2, 16)), ValueError, "aligned"),
        (dict(out=torch.zeros(3, 20)), TypeError, "out"),
        (dict(out=torch.zeros(3, 21, dtype=BF16)), ValueError, "out must be"),
        (dict(out=torch.zeros(20, dtype=BF16).expand(3, 20)), ValueError, "overlap"),
        (dict(x=torch.zeros(3, 256, dtype=BF16, requires_grad=True)), ValueError, "no backward"),
    ],
)
def test_w4_matmul_refuses(change, error, match):
    a = w4_args(**change)
    with pytest.raises(error, match=match):
        serving.w4_matmul(a.pop("x"), a.pop("codes"), a.pop("scales"), a.pop("zeros"), **a)


def cache_args(**change):
    a = dict(
        k_cache=torch.zeros(5, 2, 16, 64).to(F8), v_cache=torch.zeros(5, 2, 64, 16).to(F8),
        k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2), block_table=torch.zeros(3, 4, dtype=torch.int32),
        seq_lens=torch.ones(3, dtype=torch.int32), query_start=None,
    )
    a.update(change)
    return a


BAD_CACHE = [
    (dict(), ValueError, "on a GPU"),
    (dict(k_cache=torch.zeros(5, 2, 16, 64)), TypeError, "k_cache"),
    (dict(v_cache=torch.zeros(5, 2, 16, 64).to(F8)), ValueError, "v_cache has shape"),
    (dict(k_cache=torch.zeros(5, 2, 24, 64).to(F8)), ValueError, "page size"),
    (dict(k_cache=torch.zeros(5, 2, 16, 72).to(F8)), ValueError, "head dimension"),
    (dict(k_cache=torch.zeros(5, 2, 16, 272).to(F8)), ValueError, "head dimension"),
    (dict(k_cache=torch.zeros(0, 2, 16, 64).to(F8)), ValueError, "no cache"),
    (dict(k_scale=torch.ones(5, 1)), ValueError, "k_scale has shape"),
    (dict(v_scale=torch.ones(5, 2, dtype=BF16)), TypeError, "v_scale"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.long)), TypeError, "block_table"),
    (dict(block_table=torch.zeros(4, 3, dtype=torch.int32).t()), ValueError, "dense"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int32)), ValueError, "seq_lens has shape"),
    (dict(seq_lens=torch.ones(3, dtype=torch.long)), TypeError, "seq_lens"),
    (dict(query_start=torch.zeros(3, dtype=torch.int32)), ValueError, "query_start has shape"),
    (dict(block_table=torch.zeros(3, 2**26 + 1, dtype=torch.int32)), ValueError, "2\\^30 positions"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32)), ValueError, "query_start"),
]


@pytest.mark.parametrize("change,error,match", BAD_CACHE)
def test_cache_append_refuses(change, error, match):
    k = torch.zeros(3, 2, 64, dtype=BF16)
    with pytest.raises(error, match=match):
        serving.cache_append(k, k, **cache_args(**change))


def test_cache_append_refuses_new_tokens_that_do_not_fit():
    k = torch.zeros(3, 2, 64, dtype=BF16)
    for bad, error in ((k.float(), TypeError), (k[:, :1], ValueError), (k[0], ValueError), (k.half(), TypeError)):
        with pytest.raises(error):
            serving.cache_append(k, bad, **cache_args())


@pytest.mark.parametrize("change,error,match", BAD_CACHE)
def test_cache_attention_refuses(change, error, match):
    with pytest.raises(error, match=match):
        serving.cache_attention(torch.zeros(3, 4, 64, dtype=BF16), **cache_args(**change))


@pytest.mark.parametrize(
    "q,more,error,match",
    [
        (torch.zeros(3, 4, 64), {}, TypeError, "q has type"),
        (torch.zeros(3, 3, 64, dtype=BF16), {}, ValueError, "evenly"),
        (torch.zeros(3, 0, 64, dtype=BF16), {}, ValueError, "evenly"),
        (torch.zeros(3, 4, 80, dtype=BF16), {}, ValueError, "head dimension 80"),
        (torch.zeros(3, 4, 64, dtype=BF16), dict(window=0), ValueError, "window"),
        (torch.zeros(3, 4, 64, dtype=BF16), dict(scale=float("inf")), ValueError, "scale"),
        (torch.zeros(3, 4, 64, dtype=BF16), dict(scale=0.0), ValueError, "scale"),
        (torch.zeros(3, 4, 64, dtype=BF16), dict(out=torch.zeros(3, 4, 64)), TypeError, "out"),
        (torch.zeros(3, 4, 64, dtype=BF16), dict(out=torch.zeros(3, 64, 4, dtype=BF16).transpose(1, 2)), ValueError, "contiguous"),
        (torch.zeros(3, 4, 64, dtype=BF16, requires_grad=True), {}, ValueError, "no backward"),
    ],
)
def test_cache_attention_refuses_queries(q, more, error, match):
    with pytest.raises(error, match=match):
        serving.cache_attention(q, **cache_args(), **more)


@pytest.mark.parametrize(
    "logits,targets,top,error,match",
    [
        (torch.zeros(2, 9), torch.zeros(2, dtype=torch.long), 3, ValueError, "on a GPU"),
        (torch.zeros(2, 9).double(), torch.zeros(2, dtype=torch.long), 0, TypeError, "float64"),
        (torch.zeros(9), torch.zeros(1, dtype=torch.long), 0, ValueError, "2 dimensions"),
        (torch.zeros(2, 9), torch.zeros(2, dtype=torch.int32), 0, TypeError, "targets"),
        (torch.zeros(2, 9), torch.zeros(3, dtype=torch.long), 0, ValueError, "3 targets"),
        (torch.zeros(2, 9), torch.zeros(2, dtype=torch.long), 10, ValueError, "top_k"),
        (torch.zeros(2, 99), torch.zeros(2, dtype=torch.long), 65, ValueError, "top_k"),
        (torch.zeros(2, 9), torch.zeros(2, dtype=torch.long), -1, ValueError, "top_k"),
        (torch.zeros(2, 0), torch.zeros(2, dtype=torch.long), 0, ValueError, "vocabulary"),
        (torch.zeros(1, 1).expand(1, 2**22 + 1), torch.zeros(1, dtype=torch.long), 0, ValueError, "vocabulary"),
    ],
)
def test_token_logprobs_refuses(logits, targets, top, error, match):
    with pytest.raises(error, match=match):
        serving.token_logprobs(logits, targets, top)


def many(*shape, dtype=BF16):
    """A tensor of any size in the memory of one value."""
    return torch.zeros(1, dtype=dtype).expand(*shape)


def test_sizes_that_no_launch_can_have_are_refused():
    codes, scales, _ = serving.pack_w4(torch.zeros(16, 16, dtype=torch.uint8), torch.zeros(16, 1, dtype=BF16))
    for m, n in ((1, 2**26 + 1), (serving.MAX_TOKENS, 2**18)):
        with pytest.raises(ValueError, match="no product"):
            serving.w4_matmul(many(m, 16), codes, scales, out_features=n)
    one = dict(block_table=torch.zeros(1, 5, dtype=torch.int32), seq_lens=torch.zeros(1, dtype=torch.int32))
    one["query_start"] = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="new keys"):
        serving.cache_append(many(2**25 + 1, 2, 64), many(2**25 + 1, 2, 64), **cache_args(**one))
    with pytest.raises(ValueError, match="query rows"):
        serving.cache_attention(many(2**24 + 1, 4, 64), **cache_args(**one))
    batch = 2**21 + 1
    lens, table = torch.zeros(batch, dtype=torch.int32), torch.zeros(batch, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="heads of sequences"):
        serving.cache_attention(many(batch, 4, 64), **cache_args(block_table=table, seq_lens=lens))
    with pytest.raises(ValueError, match="rows"):
        serving.token_logprobs(many(2**24, 1), many(2**24, dtype=torch.long))


def test_pack_w4_refuses_zero_points_between_whole_numbers():
    codes, scales = torch.zeros(16, 16, dtype=torch.uint8), torch.ones(16, 1, dtype=BF16)
    assert serving.pack_w4(codes, scales, torch.full((16, 1), 3.0))[2].unique().tolist() == [3]
    with pytest.raises(ValueError, match="whole"):
        serving.pack_w4(codes, scales, torch.full((16, 1), 3.5))


def test_unpack_w4_refuses_other_sizes():
    packed, _, _ = serving.pack_w4(torch.zeros(20, 130, dtype=torch.uint8), torch.zeros(20, 2, dtype=BF16))
    assert serving.unpack_w4(packed, 20, 130).shape == (20, 130)
    for n, k in ((33, 130), (16, 130), (20, 128), (20, 257)):
        with pytest.raises(ValueError, match="packed"):
            serving.unpack_w4(packed, n, k)


def test_new_cache_refuses_sizes():
    for bad in ((0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 65, 16), (1, 1, 64, 20), (1, 1, 64, 8)):
        with pytest.raises(ValueError):
            serving.new_cache(*bad, device="cpu")


W4 = [64, 256, 3, 20, 256, 128, 0, 64, 64, 0, 64, 20, 0, 0, 0]
CACHE = [64, 64, 64, 64, 64, 64, 0, 4, 5, 2, 16, 64, 3, 4, 3]
APPEND = CACHE + [64, 128, 64, 64, 128, 64, 0, 0, 0]
ATTENTION = CACHE + [64, 256, 64, 64, 256, 64, 64, 0, 4, 0, 64, 1, 0.125, 0, 0, 0]
LOGPROBS = [64, 9, 64, 64, 64, 64, 64, 64, 0, 2, 9, 3, 0, 0, 0]


@pytest.mark.parametrize(
    "name,args,at",
    [("w4_matmul", W4, i) for i in (0, 7, 8, 10)]
    + [("cache_append", APPEND, i) for i in (0, 1, 2, 3, 4, 5, 15, 18)]
    + [("cache_attention", ATTENTION, i) for i in (0, 1, 2, 3, 4, 5, 15, 18, 21)]
    + [("token_logprobs", LOGPROBS, i) for i in (0, 2, 3, 4, 5, 6, 7)],
)
def test_tensors_without_memory_are_refused_before_a_launch(name, args, at):
    args = list(args)
    args[at] = 0
    with pytest.raises(ValueError, match="no memory"):
        getattr(_serving, name)(*args)


def test_workspaces_without_memory_are_refused_before_a_launch():
    w4 = [64, 1024, 64, 4096, 1024, 128, 0]
    assert _serving.w4_workspace(*w4) == 0
    w4[1:3] = [2048, 64]
    w4[4] = 2048
    assert _serving.w4_workspace(*w4) > 0
    with pytest.raises(ValueError, match="no memory"):
        _serving.w4_matmul(*w4, 64, 64, 0, 64, 4096, 0, 0, 0)
    assert _serving.attention_workspace(1, 1, 8, 32, 128, 0, 0, 100000) > 0
    long = [64, 64, 64, 64, 64, 64, 0, 1600, 1600, 8, 64, 128, 1, 1600, 1]
    with pytest.raises(ValueError, match="no memory"):
        _serving.cache_attention(*long, 64, 4096, 128, 64, 4096, 128, 64, 0, 32, 0, 100000, 1, 0.1, 0, 0, 0)
    assert _serving.logprob_workspace(300, 32000, 0) > 0
    with pytest.raises(ValueError, match="no memory"):
        _serving.token_logprobs(64, 32000, 64, 64, 64, 64, 0, 0, 0, 300, 32000, 0, 0, 0, 0)


def test_missing_and_empty_tensors_are_told_apart():
    """Zero points and starts may be missing; given without memory they are not that."""
    gone = torch.zeros(2, 2, 16, dtype=torch.uint8)
    gone.untyped_storage().resize_(0)
    a = w4_args(zeros=gone)
    with pytest.raises(ValueError, match="zeros has no memory"):
        serving.w4_matmul(a.pop("x"), a.pop("codes"), a.pop("scales"), a.pop("zeros"), **a)
    starts = torch.zeros(4, dtype=torch.int32)
    starts.untyped_storage().resize_(0)
    k = torch.zeros(3, 2, 64, dtype=BF16)
    with pytest.raises(ValueError, match="query_start has no memory"):
        serving.cache_append(k, k, **cache_args(query_start=starts))
    with pytest.raises(ValueError, match="query_start has no memory"):
        serving.cache_attention(torch.zeros(3, 4, 64, dtype=BF16), **cache_args(query_start=starts))


def test_tangents_are_refused():
    """In forward mode, and under torch.func.jvp, whose tensors require no gradient either."""

    def w4(**change):
        a = w4_args(**change)
        return serving.w4_matmul(a.pop("x"), a.pop("codes"), a.pop("scales"), a.pop("zeros"), **a)

    half = torch.zeros(3, 2, 64, dtype=BF16)
    calls = [
        (lambda t: w4(x=t), torch.zeros(3, 256, dtype=BF16)),
        (lambda t: w4(scales=t), torch.zeros(2, 2, 16, dtype=BF16)),
        (lambda t: w4(out=t), torch.zeros(3, 20, dtype=BF16)),
        (lambda t: serving.cache_append(t, half, **cache_args()), half),
        (lambda t: serving.cache_append(half, t, **cache_args()), half),
        (lambda t: serving.cache_append(half, half, **cache_args(k_scale=t)), torch.ones(5, 2)),
        (lambda t: serving.cache_attention(t, **cache_args()), torch.zeros(3, 4, 64, dtype=BF16)),
        (lambda t: serving.cache_attention(torch.zeros(3, 4, 64, dtype=BF16), **cache_args(v_scale=t)), torch.ones(5, 2)),
        (lambda t: serving.token_logprobs(t, torch.zeros(2, dtype=torch.long)), torch.zeros(2, 9)),
    ]
    from torch.autograd import forward_ad

    for call, t in calls:
        with forward_ad.dual_level():
            with pytest.raises(ValueError, match="tangent"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
            with pytest.raises(ValueError, match="on a GPU"):
                call(t)
        with pytest.raises(ValueError, match="tangent"):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))
        with pytest.raises(ValueError, match="on a GPU"):
            call(t)


@pytest.mark.parametrize("scale", [1e39, 3.5e38, float("nan"), -0.1])
def test_scales_past_float32_are_refused(scale):
    with pytest.raises(ValueError, match="scale"):
        serving.cache_attention(torch.zeros(3, 4, 64, dtype=BF16), **cache_args(), scale=scale)


@pytest.mark.parametrize("scale", [3.4e38, 1e-46, 1, 0.125])
def test_other_scales_are_taken(scale):
    with pytest.raises(ValueError, match="on a GPU"):
        serving.cache_attention(torch.zeros(3, 4, 64, dtype=BF16), **cache_args(), scale=scale)


# -- the build ---------------------------------------------------------------


@pytest.mark.parametrize(
    "spilled,said",
    [((0, 0), ""), ((0, 3), "second spills 3 scalar"), ((54, 0), "first spills 54 scalar"), ((), "no resource remarks")],
)
def test_build_refuses_kernels_that_spill_scalar_registers(tmp_path, spilled, said):
    import os
    import subprocess

    text = "attention.hip:9:1: warning: something else\n"
    for name, n in zip(("first", "second"), spilled):
        for line in (f"Function Name: {name}", "    SGPRs: 100", f"    SGPRs Spill: {n}", "    VGPRs Spill: 28"):
            text += f"attention.hip:1:1: remark: {line} [-Rpass-analysis=kernel-resource-usage]\n"
    log = tmp_path / "log"
    log.write_text(text)
    script = os.path.join(os.path.dirname(__file__), "..", "csrc", "scalar_spills.awk")
    r = subprocess.run(["awk", "-f", script, str(log)], capture_output=True, text=True)
    assert (r.returncode != 0) == bool(said) and said in r.stdout
    assert said or not r.stdout


# -- the diagnostic that runs them -------------------------------------------


class FakeDiag:
    def device_info(self):
        return {"device_count": 2}


class FakeServing:
    def __init__(self, **change):
        self.res = dict(
            ms_per_step=0.1, gbps=1500.0, product_gbps=1400.0, attention_gbps=2000.0, logprob_gbps=100.0,
            checked=10, verified=True, verify_failures=0, messages=[],
        )
        self.res.update(change)
        self.devices = []

    def serving_step(self, device, iters):
        self.devices.append(device)
        return self.res


def run_component(monkeypatch, fake):
    from gpud_amd.components.accelerator import diag as diag_mod
    from gpud_amd.components.base import GPUdInstance

    monkeypatch.setattr(diag_mod, "_load_diag", lambda: FakeDiag())
    monkeypatch.setattr(diag_mod, "_load_serving", lambda: fake)
    return diag_mod.ServingDiagComponent(GPUdInstance()).trigger_check()


def test_serving_component_runs_every_gpu(monkeypatch):
    fake = FakeServing()
    cr = run_component(monkeypatch, fake)
    assert cr.health == "Healthy" and fake.devices == [0, 1]
    assert cr.extra_info["gpu1.step_gbps"] == "1500"


@pytest.mark.parametrize(
    "change,said",
    [
        (dict(verified=False, verify_failures=3, messages=["logits: 3 bytes differ between two runs"]), "3 bytes differ"),
        (dict(gbps=10.0), "below floor"),
    ],
)
def test_serving_component_reports_a_sick_gpu(monkeypatch, change, said):
    cr = run_component(monkeypatch, FakeServing(**change))
    assert cr.health == "Unhealthy" and said in cr.reason
    assert cr.suggested_actions.repair_actions == ["HARDWARE_INSPECTION"]


def test_serving_component_is_registered_and_diagnosed():
    from gpud_amd.components.accelerator import diag as diag_mod
    from gpud_amd.components.base import GPUdInstance
    from gpud_amd.session.session import Session

    names = [f(GPUdInstance()).name for f in diag_mod.init_funcs()]
    assert diag_mod.NAME_SERVING in names
    assert diag_mod.NAME_SERVING in Session.DIAG_COMPONENTS
