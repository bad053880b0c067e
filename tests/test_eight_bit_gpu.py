"""A cache in 8 bits and trees of drafted tokens on the GPU, each operation against its plain form in 64 bits."""

import math

import pytest
import torch

import plain_cache as plain
from distie_amd.kernels.interface import EightBitCache

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from distie_amd.kernels.hip_ops import HipOps

    return HipOps("cuda:0")


def empty_cache(pages, kv_heads, page, dim, fill=0x7F):
    codes = lambda *shape: torch.full(shape, fill, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    powers = lambda: torch.full((pages, kv_heads, page), 3, dtype=torch.uint8, device="cuda")
    return EightBitCache(codes(pages, kv_heads, page, dim), codes(pages, kv_heads, dim, page), powers(), powers())


def by_slot(cache):
    """(k, v) values float64 [pages * P, KH, D], (k, v) bytes [pages * P, KH]"""
    k, v = cache.k.cpu().double().transpose(1, 2), cache.v.cpu().double().permute(0, 3, 1, 2)
    kb, vb = (x.cpu().transpose(1, 2).int() for x in (cache.k_scale, cache.v_scale))
    k, v = (torch.ldexp(x, b[..., None] - 127) for x, b in ((k, kb), (v, vb)))
    return (k.flatten(0, 1), v.flatten(0, 1)), (kb.flatten(0, 1), vb.flatten(0, 1))


def half_step(x, byte):
    """Half the distance between codes around x: 2^-4 of its power of two, and no less than half of 2^-9."""
    unit = torch.exp2(byte.double() - 127)[..., None]
    return torch.exp2(torch.floor(torch.log2((x.abs() / unit).clamp(min=2.0 ** -6)))) * unit * 2.0 ** -4


# ------------------------------------------------------------------------------------------------------- write and read
@pytest.mark.parametrize("H, KH, D, P, act, rotary, past, new", [
    (12, 2, 128, 16, BF16, 128, [500, 0, 2047], [1, 1, 1]),
    (28, 4, 128, 16, BF16, 128, [0, 33], [67, 5]),
    (28, 4, 128, 16, F32, 128, [13], [50]),
    (14, 2, 64, 32, BF16, 64, [0, 7, 31, 100000], [33, 1, 2, 16]),
    (4, 4, 96, 16, BF16, 96, [15], [18]),
    (8, 1, 256, 64, BF16, 256, [120000], [70]),
    (8, 2, 128, 16, BF16, 32, [5], [21]),                   # part of a head is rotated
    (8, 2, 128, 16, BF16, 0, [5], [21]),                    # nothing is
    (3, 1, 40, 8, F32, 40, [3, 0], [9, 4]),
    (6, 3, 10, 5, BF16, 6, [3, 0], [9, 4]),
    (2, 2, 80, 24, BF16, 80, [1], [47]),
    (32, 8, 128, 16, BF16, 128, [0, 40, 3], [130, 4, 4]),
])
def test_write_and_read(ops, H, KH, D, P, act, rotary, past, new):
    batch = plain.Batch(past, new, P, "cuda", seed=D + P)
    gen = torch.Generator().manual_seed(7)
    T = sum(new)
    x = torch.randn(T, H + 2 * KH, D, generator=gen) * torch.exp(torch.randn(T, H + 2 * KH, 1, generator=gen) * 2)
    x[0, H, :] = 0                                           # a key of zeros
    x[-1, H + KH, :] *= 1e-30
    qkv = x.view(T, -1).to(act)
    x = qkv.view(x.shape).double()
    freq = (10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))).float() if rotary else None
    cache = empty_cache(batch.pages, KH, P, D)
    before, bytes_before = by_slot(cache)
    given = qkv.cuda()
    q = ops.rope_kv_write_e4m3(given, batch.meta, 0, cache, None if freq is None else freq.cuda(), H, KH, D, True)
    assert torch.equal(given.cpu(), qkv)
    turned = plain.rotated(x[:, :H + KH], batch.positions, freq) if rotary else x[:, :H + KH]
    # cosine, sine, two products and a sum, each rounded once
    half = rotary // 2
    near = torch.zeros_like(turned)
    both = x[:, :H + KH, :half].abs() + x[:, :H + KH, half:rotary].abs()
    near[..., :half] = near[..., half:rotary] = both * 3 * 2.0 ** -24
    bound = near[:, :H] + (2.0 ** -8 * (turned[:, :H].abs() + near[:, :H]) if act == BF16 else 0)
    assert q.dtype == act and ((q.cpu().double().view(T, H, D) - turned[:, :H]).abs() <= bound).all()

    (k, v), (kb, vb) = by_slot(cache)
    slots = batch.slots.long()
    want_v, want_vb = plain.quantised(x[:, H + KH:])
    assert torch.equal(vb[slots].long(), want_vb) and torch.equal(v[slots], want_v)
    key, slack = turned[:, H:], near[:, H:]
    for t in range(T):
        for h in range(KH):
            allowed = {plain.power_of(key[t, h].abs() + slack[t, h]), plain.power_of((key[t, h].abs() - slack[t, h]).clamp(min=0))}
            assert int(kb[slots[t], h]) in allowed
    assert ((k[slots] - key).abs() <= half_step(key, kb[slots]) + slack).all()
    others = torch.ones(len(k), dtype=torch.bool)
    others[slots] = False
    for now, then in ((k, before[0]), (v, before[1]), (kb, bytes_before[0]), (vb, bytes_before[1])):
        assert torch.equal(now[others].nan_to_num(-1.0), then[others].nan_to_num(-1.0))         # no other place was written

    for dtype in (F32, BF16):
        got = ops.read_kv_e4m3(cache, batch.meta.groups[0].slots, dtype)
        assert torch.equal(got[0].cpu().double(), k[slots].to(dtype).double()) and torch.equal(got[1].cpu().double(), v[slots].to(dtype).double())
    outside = torch.tensor([-1, batch.pages * P, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    assert all(float(t.abs().max()) == 0 for t in ops.read_kv_e4m3(cache, outside, F32))


def test_write_takes_slices_views_and_no_write(ops):
    from distie_amd.kernels.hip_ops import PartialSums

    H, KH, D, P = 12, 2, 128, 16
    batch = plain.Batch([3, 20], [1, 9], P, "cuda")
    freq = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().cuda()
    gen = torch.Generator(device="cuda").manual_seed(1)
    parts = torch.randn(5, 10, (H + 2 * KH) * D, generator=gen, device="cuda")
    whole = parts[0].clone()
    for p in parts[1:]:
        whole += p
    caches = [empty_cache(batch.pages, KH, P, D) for _ in range(4)]
    run = lambda x, cache, write=True: ops.rope_kv_write_e4m3(x, batch.meta, 0, cache, freq, H, KH, D, write)
    q = run(whole, caches[0])
    sliced = run(PartialSums(parts, F32), caches[1])
    wide = torch.randn(10, (H + 2 * KH) * D + 24, generator=gen, device="cuda")
    wide[:, 8:-16] = whole
    view = run(wide[:, 8:-16], caches[2])
    kept = run(whole, caches[3], write=False)
    for other in (sliced, view, kept):
        assert torch.equal(q, other)
    for name in ("k", "v", "k_scale", "v_scale"):
        first = getattr(caches[0], name).view(torch.uint8)
        assert torch.equal(first, getattr(caches[1], name).view(torch.uint8)) and torch.equal(first, getattr(caches[2], name).view(torch.uint8))
        assert torch.equal(getattr(caches[3], name).view(torch.uint8), getattr(empty_cache(batch.pages, KH, P, D), name).view(torch.uint8))


@pytest.mark.parametrize("D", [128, 10])
def test_write_keeps_what_is_not_finite_and_the_largest(ops, D):
    H = KH = 1
    batch = plain.Batch([0], [6], 16, "cuda")
    x = torch.ones(6, 3, D)
    x[0, 2, 0], x[0, 2, 1], x[0, 2, 2] = math.inf, -math.inf, math.nan
    x[1, 2, 0], x[1, 2, 1] = torch.finfo(F32).max, -torch.finfo(F32).max
    x[2, 2, 0] = 2.0 ** -149                                  # beside ones
    x[3, 2] = 2.0 ** -149
    x[4, 2] = math.nan
    x[5, 2, 0], x[5, 2, 1] = 448 * 2.0 ** -20, 449 * 2.0 ** -20
    x[5, 2, 2:] = 0
    cache = empty_cache(batch.pages, KH, 16, D)
    ops.rope_kv_write_e4m3(x.view(6, -1).cuda(), batch.meta, 0, cache, None, H, KH, D, True)
    want, bytes_ = plain.quantised(x[:, 2:].double())
    (_, v), (_, vb) = by_slot(cache)
    slots = batch.slots.long()
    assert torch.equal(vb[slots].long(), bytes_)
    assert torch.equal(v[slots].isnan(), want.isnan()) and torch.equal(v[slots].nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("M, C, I, H, KH, D, biased", [(1, 1024, 2816, 16, 2, 64, True), (8, 1536, 8960, 12, 2, 128, True), (3, 2048, 1056, 8, 1, 16, False)])
def test_the_rows_behind_a_layers_end(ops, M, C, I, H, KH, D, biased):
    """They are the bits of the rotated and written form at position 0, where nothing turns; written from there, those of the same rows
    from anywhere else."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    rand = lambda *shape, scale=1.0: (torch.randn(*shape, generator=gen, device="cuda") * scale).to(BF16)
    N = (H + 2 * KH) * D
    mixed, residual = rand(M, H * D), rand(M, C).float()
    w_o, w_gu, w_d, w_qkv = rand(C, H * D, scale=D ** -0.5 / 4), rand(2 * I, C, scale=C ** -0.5), rand(C, I, scale=I ** -0.5), rand(N, C, scale=C ** -0.5)
    for weight, kinds in ((w_o, {}), (w_gu, {"gated": True}), (w_d, {}), (w_qkv, {"rotary": (H, KH, D)})):
        ops.prepare_linear(weight, **kinds)
    norm, bias = rand(C).float(), rand(N).float() if biased else None
    freq = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().cuda()
    start, batch = plain.Batch([0] * M, [1] * M, 16, "cuda"), plain.Batch([40 * i for i in range(M)], [1] * M, 16, "cuda")
    ops.captured = True
    try:
        tail = lambda meta: ops.layer_tail(meta, residual, mixed, w_o, norm, 1e-5, w_gu, w_d)
        k, v = (torch.zeros(start.pages, KH, *shape, dtype=BF16, device="cuda") for shape in ((16, D), (D, 16)))
        hidden, want = tail(start.meta).finish_into(norm, 1e-5, w_qkv, bias, start.meta, 0, k, v, freq, H, KH, D, False)
        again, rows = tail(batch.meta).finish_rows(norm, 1e-5, w_qkv, bias, batch.meta, H, KH, D)
        assert torch.equal(hidden, again) and torch.equal(rows, want) and rows.shape == (M, N)
        assert tail(batch.meta).finish_rows(norm, 1e-5, w_qkv.clone(), bias, batch.meta, H, KH, D) is None            # no packed copy
    finally:
        ops.captured = False
    caches = [empty_cache(batch.pages, KH, 16, D) for _ in range(2)]
    q = [ops.rope_kv_write_e4m3(x, batch.meta, 0, c, freq, H, KH, D, True) for x, c in zip((rows, rows.clone()), caches)]
    assert torch.equal(*q) and torch.equal(*(c.k.view(torch.uint8) for c in caches)) and torch.equal(*(c.v.view(torch.uint8) for c in caches))


def layer_end(ops, M, C, I, H, KH, D, seed=1):
    """-> (rows of the next layer's q/k/v product for a bias and further arguments of `finish_rows`, the product's weight and norm)"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape, scale=1.0: (torch.randn(*shape, generator=gen, device="cuda") * scale).to(BF16)
    mixed, residual = rand(M, H * D), rand(M, C).float()
    w_o, w_gu, w_d, w_qkv = rand(C, H * D, scale=D ** -0.5 / 4), rand(2 * I, C, scale=C ** -0.5), rand(C, I, scale=I ** -0.5), rand((H + 2 * KH) * D, C, scale=C ** -0.5)
    for weight, kinds in ((w_o, {}), (w_gu, {"gated": True}), (w_d, {}), (w_qkv, {"rotary": (H, KH, D)})):
        ops.prepare_linear(weight, **kinds)
    norm, batch = rand(C).float(), plain.Batch([40 * i for i in range(M)], [1] * M, 16, "cuda")

    def rows(bias, *more):
        ops.captured = True
        try:
            return ops.layer_tail(batch.meta, residual, mixed, w_o, norm, 1e-5, w_gu, w_d).finish_rows(norm, 1e-5, w_qkv, bias, batch.meta, H, KH, D, *more)
        finally:
            ops.captured = False

    return rows, w_qkv, norm, batch


@pytest.mark.parametrize("M", [1, 8])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_the_rows_behind_a_layers_end_stand_for_themselves(ops, M, value):
    """What is not finite in one column of q or k is not in the column that a rotation would turn it with."""
    H, KH, D = 12, 2, 128
    rows, w_qkv, _, _ = layer_end(ops, M, 1536, 8960, H, KH, D)
    bias = torch.randn((H + 2 * KH) * D, generator=torch.Generator().manual_seed(3)).cuda()
    want = rows(bias)[1]
    odd = torch.tensor([5, 3 * D + 70, (H + 1) * D + 127, (H + KH) * D + 1], device="cuda")          # of q, of k, of v
    bias[odd] = value
    got = rows(bias)[1]
    whole = torch.ones(bias.shape[0], dtype=torch.bool, device="cuda")
    whole[odd] = False
    assert not got[:, odd].isfinite().any() and torch.equal(got[:, whole], want[:, whole])


@pytest.mark.parametrize("M, C, I, H, KH, D, biased", [(1, 1024, 2816, 16, 2, 64, True), (8, 1536, 8960, 12, 2, 128, True), (3, 2048, 1056, 8, 1, 16, False)])
def test_the_rows_behind_a_layers_end_are_float32_sums(ops, M, C, I, H, KH, D, biased):
    """As `linear` hands them on to the write: keys and values are rounded once, to codes, and q once, behind its rotation. The norm in front of
    the product is rounded to bfloat16; where its float32 value (off by at most 20 roundings: a mean of squares of 30 steps, halved by the
    root, the root, two products) may have been rounded to either neighbour, their distance is part of the bound. The sums: a wave takes C / 256
    products of 32 terms, eight waves and a bias are added up, a rounding for each."""
    from distie_amd.kernels.hip_ops import PartialSums

    rows, w_qkv, norm, batch = layer_end(ops, M, C, I, H, KH, D, seed=M + 10)
    N = (H + 2 * KH) * D
    bias = torch.randn(N, generator=torch.Generator().manual_seed(3)).cuda() if biased else None
    hidden, sums = rows(bias, True)
    assert isinstance(sums, PartialSums) and sums.dtype == BF16 and tuple(sums.shape) == (M, N)
    got = sums.data.double().sum(0).cpu()
    h = hidden.double().cpu()
    x = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + 1e-5) * norm.double().cpu()
    low, high = ((x * (1 + e)).to(BF16).double() for e in (-20 * 2.0 ** -24, 20 * 2.0 ** -24))
    w, b = w_qkv.double().cpu(), 0 if bias is None else bias.double().cpu()
    x, roundings = x.to(BF16).double(), C // 256 * 33 + 9
    bound = (high - low).abs() @ w.abs().T + roundings * 2.0 ** -24 * (x.abs() @ w.abs().T + (0 if bias is None else b.abs()))
    away = (got - (x @ w.T + b)).abs()
    assert (away <= bound).all(), float((away / bound).max())
    assert ((got.to(BF16).double() - (x @ w.T + b)).abs() > bound).any()          # (rows rounded to bfloat16 would not pass)
    assert torch.equal(rows(bias)[1], ops.dense(sums)) and torch.equal(ops.dense(sums).cpu(), got.float().to(BF16))
    # written from there
    freq = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().cuda()
    caches = [empty_cache(batch.pages, KH, 16, D) for _ in range(2)]
    q = [ops.rope_kv_write_e4m3(r, batch.meta, 0, c, freq, H, KH, D, True) for r, c in zip((sums, sums.data.sum(0)), caches)]
    assert q[0].dtype == BF16 and torch.equal(q[0], q[1].to(BF16))
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(*(getattr(c, name).view(torch.uint8) for c in caches))
    (_, v), (_, vb) = by_slot(caches[0])
    want, want_vb = plain.quantised(got.view(M, -1, D)[:, H + KH:])
    assert torch.equal(vb[batch.slots.long()].long(), want_vb) and torch.equal(v[batch.slots.long()], want)


# -------------------------------------------------------------------------------------------------------------- attention
def check_attention(ops, H, KH, D, batch, act, kind, window, seed=0, garbage=math.nan, view=False):
    cache, keys, values = plain.random_cache(batch, KH, D, kind, seed, "cuda", garbage)
    gen = torch.Generator().manual_seed(seed + 1)
    T = batch.meta.num_tokens
    q = (1.5 * torch.randn(T, H * D, generator=gen)).to(act)
    given = q.cuda()
    if view:
        wide = torch.full((T, H * D + 64), math.nan, dtype=act, device="cuda")
        wide[:, 16:16 + H * D] = given
        given = wide[:, 16:16 + H * D]
    scale = D ** -0.5
    call = ops.paged_attention_e4m3 if batch.sees is None else ops.tree_attention
    got = call(given, batch.meta, 0, cache, H, KH, D, scale, window)
    want, sizes, scores, most = plain.attended(q.double().view(T, H, D), batch, keys, values, KH, scale, window)
    bound = plain.attention_bound(want, sizes, scores, most, D, act)
    away = (got.cpu().double().view(T, H, D) - want).abs()
    assert got.dtype == act and got.isfinite().all()
    assert (away <= bound).all(), f"{float((away / bound).max())} times the bound"
    return got


HEADS = [(12, 2, 128, 16), (28, 4, 128, 32), (14, 2, 64, 16), (4, 4, 96, 16), (8, 1, 256, 64), (5, 5, 32, 48), (40, 1, 64, 16), (3, 1, 40, 8), (6, 2, 80, 16), (2, 1, 48, 5)]


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("H, KH, D, P", HEADS)
def test_attention_single_tokens(ops, H, KH, D, P, act):
    past = [0, 1, 15, 16, 62, 63, 64, 65, 517, 1300]
    check_attention(ops, H, KH, D, plain.Batch(past, [1] * len(past), P, "cuda", table_rows=True), act, "e4m3", None)


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("H, KH, D, P", HEADS)
def test_attention_portions(ops, H, KH, D, P, act):
    check_attention(ops, H, KH, D, plain.Batch([0, 37, 200, 5], [70, 3, 131, 1], P, "cuda"), act, "e4m3", None)


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("window", [1, 16, 50, 64, 129])
def test_attention_windows(ops, window, act):
    for past, new in ([0, 15, 200, 511], [1, 1, 1, 1]), ([0, 100, 300], [90, 1, 40]):
        batch = plain.Batch(past, new, 16, "cuda", window=window)
        check_attention(ops, 12, 2, 128, batch, act, "e4m3", window)


def test_single_tokens_beside_portions(ops):
    check_attention(ops, 28, 4, 128, plain.Batch([900, 0, 333, 40, 0, 2100], [1, 150, 1, 66, 1, 1], 16, "cuda", table_rows=True), BF16, "e4m3", None)
    check_attention(ops, 28, 4, 128, plain.Batch([900, 0, 333], [1, 150, 1], 16, "cuda", window=100), BF16, "e4m3", 100)


def test_attention_of_one_long_context(ops):
    check_attention(ops, 28, 4, 128, plain.Batch([20001], [1], 16, "cuda"), BF16, "e4m3", None)
    check_attention(ops, 12, 2, 128, plain.Batch([9000, 1], [3, 1], 16, "cuda"), F32, "e4m3", None)


@pytest.mark.parametrize("act", [BF16, F32])
def test_attention_of_a_view(ops, act):
    check_attention(ops, 12, 2, 128, plain.Batch([30, 7], [1, 5], 16, "cuda"), act, "e4m3", None, view=True)
    check_attention(ops, 12, 2, 128, plain.Batch([300, 700], [1, 1], 16, "cuda"), act, "e4m3", None, view=True)


def tree_batch(past, new, page, seed, positions=True, **more):
    gen = torch.Generator().manual_seed(seed)
    trees = [plain.random_tree(n, gen) for n in new]
    where = torch.cat([p + d for p, (_, d) in zip(past, trees)]).int()
    return plain.Batch(past, new, page, "cuda", seed=seed, tree=[s for s, _ in trees], positions=where, **more)


KINDS = [(BF16, "e4m3"), (BF16, BF16), (F32, "e4m3"), (F32, F32)]


@pytest.mark.parametrize("act, kind", KINDS)
@pytest.mark.parametrize("H, KH, D, P", HEADS)
def test_trees(ops, H, KH, D, P, act, kind):
    check_attention(ops, H, KH, D, tree_batch([0, 1, 60, 64, 333], [7, 1, 12, 64, 65], P, seed=D, table_rows=True), act, kind, None)


@pytest.mark.parametrize("act, kind", KINDS)
@pytest.mark.parametrize("past, new", [([300], [7]), ([0], [1]), ([0, 0], [200, 3]), ([5000, 17], [61, 61]), ([1000] * 3, [130, 129, 1])])
def test_trees_of_many_sizes(ops, past, new, act, kind):
    check_attention(ops, 28, 4, 128, tree_batch(past, new, 16, seed=5), act, kind, None)


@pytest.mark.parametrize("act, kind", KINDS)
@pytest.mark.parametrize("window", [1, 3, 17, 100])
def test_trees_under_a_window(ops, window, act, kind):
    check_attention(ops, 12, 2, 128, tree_batch([0, 40, 250], [20, 70, 9], 16, seed=9, window=window), act, kind, window)


@pytest.mark.parametrize("act, kind", KINDS)
@pytest.mark.parametrize("D, P", [(128, 16), (40, 8)])
def test_tree_tokens_that_see_nothing(ops, D, P, act, kind):
    """Without a context and with no bit set a token's result is zero, whatever the others see."""
    batch = tree_batch([0, 0, 30], [9, 1, 4], P, seed=2)
    for b, row in ((0, 0), (0, 5), (1, 0), (2, 3)):
        batch.sees[b][row] = False
        batch.meta.tree[int(batch.cu[b]) + row] = 0
    got = check_attention(ops, 6, 2, D, batch, act, kind, None)
    assert float(got[0].abs().max()) == float(got[5].abs().max()) == float(got[9].abs().max()) == 0


@pytest.mark.parametrize("act, kind", KINDS)
@pytest.mark.parametrize("D, P", [(128, 16), (256, 16), (40, 8)])
@pytest.mark.parametrize("new", [7, 70])
def test_what_a_tree_token_does_not_see_is_not_in_its_result(ops, D, P, new, act, kind):
    """NaN and infinities in drafted keys and values reach those tokens that see them, and no other."""
    H, KH = 6, 2
    batch = tree_batch([37, 0], [new, 5], P, seed=3)
    cache, keys, values = plain.random_cache(batch, KH, D, kind, 4, "cuda")
    k, v = (cache.k, cache.v) if kind == "e4m3" else cache
    entries, bad = batch.entries(0), {2: math.nan, 4: math.nan if kind == "e4m3" else math.inf, new - 1: math.nan}
    for i, value in bad.items():
        page, at = divmod(int(entries[37 + i]), P)
        if i != 4:
            k[page, :, at, 3] = value
        v[page, :, 5, at] = value
    gen = torch.Generator().manual_seed(8)
    q = torch.randn(batch.meta.num_tokens, H * D, generator=gen).to(act)
    got = ops.tree_attention(q.cuda(), batch.meta, 0, cache, H, KH, D, D ** -0.5, None).cpu().double().view(-1, H, D)
    want, sizes, scores, most = plain.attended(q.double().view(-1, H, D), batch, keys, values, KH, D ** -0.5)
    bound = plain.attention_bound(want, sizes, scores, most, D, act)
    for t in range(batch.meta.num_tokens):
        sees = batch.sees[0][t] if t < new else torch.zeros(new, dtype=torch.bool)
        if any(bool(sees[i]) for i in bad if i != 4):
            assert got[t].isnan().all(), t
        elif new > 4 and bool(sees[4]):
            assert not got[t, :, 5].isfinite().any(), t
            rest = torch.arange(D) != 5
            assert ((got[t] - want[t]).abs() <= bound[t])[:, rest].all(), t
        else:
            assert ((got[t] - want[t]).abs() <= bound[t]).all(), t


def test_entries_beyond_four_gigabytes(ops):
    """The requests' pages lie at the far end of a cache of more than 2^32 values."""
    H, KH, D, P = 4, 1, 128, 16
    near = plain.Batch([100, 40], [1, 1], P, "cuda")
    cache, keys, values = plain.random_cache(near, KH, D, "e4m3", 0, "cuda")
    far = 2 ** 32 // (KH * P * D) + 3
    codes = lambda *shape: torch.empty(far + near.pages, *shape, dtype=torch.uint8, device="cuda")
    big = EightBitCache(codes(KH, P, D).view(torch.float8_e4m3fn), codes(KH, D, P).view(torch.float8_e4m3fn), codes(KH, P), codes(KH, P))
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(big, name).view(torch.uint8)[far:] = getattr(cache, name).view(torch.uint8)
    q = torch.randn(2, H * D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    want = ops.paged_attention_e4m3(q, near.meta, 0, cache, H, KH, D, 0.1, None)
    table = near.meta.groups[0].block_table
    table[table >= 0] += far
    near.meta.scratch.clear()
    assert torch.equal(ops.paged_attention_e4m3(q, near.meta, 0, big, H, KH, D, 0.1, None), want)
    # the slots of such a cache pass 2^31 places only with far more pages; their bytes pass 2^32 here
    slots = near.meta.groups[0].slots
    k, v = ops.read_kv_e4m3(cache, slots, F32)
    slots += far * P
    for got, held in zip(ops.read_kv_e4m3(big, slots, F32), (k, v)):
        assert torch.equal(got, held)
    qkv = torch.randn(2, (H + 2 * KH) * D, generator=torch.Generator().manual_seed(2)).cuda()
    ops.rope_kv_write_e4m3(qkv, near.meta, 0, big, None, H, KH, D, True)
    k, v = ops.read_kv_e4m3(big, slots, F32)
    want, _ = plain.quantised(qkv.cpu().double().view(2, -1, D)[:, H:])
    assert torch.equal(torch.cat([k, v], 1).cpu().double(), want)


@pytest.mark.parametrize("act, H, past, new", [(BF16, 12, [100, 30], [1, 1]), (F32, 12, [100, 30], [1, 9]), (BF16, 12, [100], [130])])
@pytest.mark.parametrize("P", [16, 8])
def test_a_window_does_not_let_through_what_lies_before_it(ops, act, H, past, new, P):
    """NaN among the entries that a window has passed, on pages that other tokens still see, reaches only those."""
    KH, D, window = 2, 128, 20
    batch = plain.Batch(past, new, P, "cuda", seed=1)
    cache, keys, values = plain.random_cache(batch, KH, D, "e4m3", 2, "cuda")
    for b, p in enumerate(past):
        page, at = divmod(int(batch.entries(b)[p - window // 2 - 4]), P)
        cache.k.view(torch.uint8)[page, :, at, 3] = cache.v.view(torch.uint8)[page, :, 5, at] = 0x7F
        page, at = divmod(int(batch.entries(b)[p - window]), P)
        cache.k.view(torch.uint8)[page, :, at, 3] = cache.v.view(torch.uint8)[page, :, 5, at] = 0x7F
    q = torch.randn(sum(new), H * D, generator=torch.Generator().manual_seed(3)).to(act)
    got = ops.paged_attention_e4m3(q.cuda(), batch.meta, 0, cache, H, KH, D, 0.1, window).cpu().double().view(-1, H, D)
    want, sizes, scores, most = plain.attended(q.double().view(-1, H, D), batch, keys, values, KH, 0.1, window)
    bound = plain.attention_bound(want, sizes, scores, most, D, act)
    for t in range(sum(new)):
        b = int(batch.request[t])
        if int(batch.positions[t]) - (past[b] - window // 2 - 4) < window:
            assert got[t].isnan().all(), t
        else:
            assert ((got[t] - want[t]).abs() <= bound[t]).all(), t


@pytest.mark.parametrize("act, kind", KINDS)
@pytest.mark.parametrize("P", [16, 8])
def test_requests_without_tokens_and_steps_without_requests(ops, P, act, kind):
    if kind == "e4m3":
        check_attention(ops, 12, 2, 128, plain.Batch([40, 7, 0, 300], [0, 5, 0, 1], P, "cuda"), act, kind, None)
        check_attention(ops, 12, 2, 128, plain.Batch([40, 7, 0], [0, 200, 0], P, "cuda"), act, kind, None)
    none = torch.zeros(0, 0, dtype=torch.bool)
    tree = [none, plain.random_tree(9, torch.Generator().manual_seed(1))[0], none]
    check_attention(ops, 12, 2, 128, plain.Batch([40, 7, 0], [0, 9, 0], P, "cuda", tree=tree), act, kind, None)
    empty = plain.Batch([7], [1], P, "cuda").meta
    empty.num_tokens = empty.num_requests = 0
    for name in ("positions", "token_request", "kv_len"):
        setattr(empty, name, getattr(empty, name)[:0])
    empty.cu_q, empty.host_cu_q, empty.host_past = empty.cu_q[:1], empty.host_cu_q[:1], empty.host_past[:0]
    empty.groups[0].slots, empty.groups[0].block_table = empty.groups[0].slots[:0], empty.groups[0].block_table[:0]
    cache, _, _ = plain.random_cache(plain.Batch([7], [1], P), 2, 128, kind, 0, "cuda", 0.0)
    q = torch.zeros(0, 12 * 128, dtype=act, device="cuda")
    if kind == "e4m3":
        assert ops.paged_attention_e4m3(q, empty, 0, cache, 12, 2, 128, 1.0, None).shape == (0, 12 * 128)
        assert ops.rope_kv_write_e4m3(torch.zeros(0, 16 * 128, dtype=act, device="cuda"), empty, 0, cache, None, 12, 2, 128, True).shape == (0, 12 * 128)
        assert ops.read_kv_e4m3(cache, empty.groups[0].slots, F32)[0].shape == (0, 2, 128)
    empty.tree = torch.zeros(0, 1, dtype=torch.int64, device="cuda")
    assert ops.tree_attention(q, empty, 0, cache, 12, 2, 128, 1.0, None).shape == (0, 12 * 128)


def test_a_float32_portion_of_many_column_tiles(ops):
    """More tiles of columns than a grid's second axis holds (65,535)."""
    H, KH, D, T = 64, 64, 32, 16400
    batch = plain.Batch([0], [T], 16, "cuda", window=3)
    cache, keys, values = plain.random_cache(batch, KH, D, "e4m3", 0, "cuda", 0.0)
    q = torch.randn(T, H * D, generator=torch.Generator().manual_seed(1))
    got = ops.paged_attention_e4m3(q.cuda(), batch.meta, 0, cache, H, KH, D, 0.2, 3).cpu().double().view(T, H, D)
    slots = batch.entries(0)
    k, v = keys[slots].transpose(0, 1), values[slots].transpose(0, 1)                    # [H, T, D]
    q = q.double().view(T, H, D).transpose(0, 1)
    scores = torch.stack([(q[:, i:] * k[:, :T - i]).sum(-1) if not i else
                          torch.cat([torch.full((H, i), -math.inf, dtype=torch.float64), (q[:, i:] * k[:, :T - i]).sum(-1)], 1) for i in range(3)], -1) * 0.2
    w = torch.softmax(scores, -1)
    near = torch.stack([torch.cat([torch.zeros(H, i, D, dtype=torch.float64), v[:, :T - i]], 1) for i in range(3)], 2)
    want = (w[..., None] * near).sum(2).transpose(0, 1)
    sizes = (w[..., None] * near.abs()).sum(2).transpose(0, 1)
    largest = (q.norm(dim=-1).max() * k.norm(dim=-1).max() * 0.2)
    assert ((got - want).abs() <= plain.attention_bound(want, sizes, largest, 3, D, F32)).all()


@pytest.mark.parametrize("new", [[1, 1], [9, 40]])
@pytest.mark.parametrize("by", [-80, 90])
def test_float32_queries_far_from_one(ops, new, by):
    """Queries times a power of two and a scale over it: the same scores, so the same bits (80 under the lowest bit of a query of 2^-10
    is 2^-114, which every type here holds)."""
    H, KH, D = 12, 2, 128
    batch = plain.Batch([300, 70], new, 16, "cuda")
    cache, _, _ = plain.random_cache(batch, KH, D, "e4m3", 3, "cuda", math.nan)
    q = torch.randn(sum(new), H * D, generator=torch.Generator().manual_seed(4))
    q = torch.where(q.abs() < 2.0 ** -10, torch.zeros(()), q).cuda()
    near = ops.paged_attention_e4m3(q, batch.meta, 0, cache, H, KH, D, 2.0 ** -4, None)
    far = ops.paged_attention_e4m3(q * 2.0 ** by, batch.meta, 0, cache, H, KH, D, 2.0 ** (-4 - by), None)
    assert near.isfinite().all() and torch.equal(near, far)


@pytest.mark.parametrize("kind", ["e4m3", BF16])
@pytest.mark.parametrize("H, KH, D, past, new, window", [
    (80, 1, 32, [190], [60], None),                         # entries that every token sees, not cut
    (12, 2, 128, [3000, 20], [100, 90], 1000),              # cut, behind a window
    (28, 4, 128, [1500, 0, 700], [130, 1, 77], None),
    (28, 4, 64, [2000, 1999, 30], [90, 90, 200], None),
    (6, 2, 256, [900, 64], [80, 129], 500),
])
def test_many_columns(ops, H, KH, D, past, new, window, kind):
    tree = tree_batch(past, new, 16, seed=9, window=window)
    check_attention(ops, H, KH, D, tree, BF16, kind, window)
    if kind == "e4m3":
        check_attention(ops, H, KH, D, plain.Batch(past, new, 16, "cuda", window=window), BF16, kind, window)


@pytest.mark.parametrize("new", [[1, 1, 1], [1, 0, 40]])
def test_a_step_described_as_larger_than_it_is(ops, new):
    """`max_q` and `max_kv` are bounds: a description made for a larger step gives the same."""
    batch = plain.Batch([1500, 30, 700], new, 16, "cuda", spare=200)
    batch.meta.max_q, batch.meta.max_kv, batch.meta.all_decode = 700, 2300, False
    check_attention(ops, 28, 4, 128, batch, BF16, "e4m3", None)
    check_attention(ops, 12, 2, 128, batch, F32, "e4m3", None)


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("before, after", [(([100, 40], [3, 4]), ([100, 40], [3, 200])), (([100, 40], [3, 200]), ([4000, 3500], [3, 200])),
                                           (([900], [70]), ([900, 20, 3000], [80, 30, 1]))])
def test_a_description_that_changes_between_calls(ops, act, before, after):
    """More tokens a request, longer contexts, more requests than in the call before: nothing of that call's launches or parts is kept."""
    batch, then = plain.Batch(*before, 16, "cuda"), plain.Batch(*after, 16, "cuda")
    batch.meta.max_kv = then.meta.max_kv = 6000
    cu_q = batch.meta.host_cu_q
    check_attention(ops, 12, 2, 128, batch, act, "e4m3", None)
    scratch, whole = batch.meta.scratch, dict(then.meta.__dict__)
    batch.meta.__dict__.update(whole)
    batch.meta.scratch, then.meta = scratch, batch.meta
    if before[1] == after[1]:
        batch.meta.host_cu_q = cu_q
    check_attention(ops, 12, 2, 128, then, act, "e4m3", None)


def test_more_requests_than_a_wave_has_lanes(ops):
    new = [40 + 3 * (i % 7) for i in range(70)] + [0, 33, 0]
    past = [(37 * i) % 300 for i in range(73)]
    check_attention(ops, 32, 4, 32, plain.Batch(past, new, 16, "cuda", table_rows=True), BF16, "e4m3", None)


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32 + 5, 2 ** 63])
def test_windows_that_hold_every_position(ops, window):
    batch = plain.Batch([300, 7], [1, 30], 16, "cuda")
    cache, _, _ = plain.random_cache(batch, 2, 128, "e4m3", 3, "cuda", 0.0)
    q = torch.randn(31, 12 * 128, device="cuda").bfloat16()
    call = lambda w: ops.paged_attention_e4m3(q, batch.meta, 0, cache, 12, 2, 128, 0.1, w)
    assert torch.equal(call(window), call(None))


def test_runs_of_one_call_are_the_same(ops):
    batch = plain.Batch([700, 3000], [1, 1], 16, "cuda")
    first = check_attention(ops, 28, 4, 128, batch, BF16, "e4m3", None)
    for _ in range(3):
        assert torch.equal(check_attention(ops, 28, 4, 128, batch, BF16, "e4m3", None), first)


# ------------------------------------------------------------------------------------------------------------------ keep
@pytest.mark.parametrize("dtype, shape, axis", [(BF16, (4, 16, 32), 3), (BF16, (4, 32, 16), 4), (F32, (3, 5, 6), 3), (torch.uint8, (4, 16), 3),
                                                (torch.uint8, (2, 16, 48), 3), (torch.uint8, (2, 40, 8), 4), (BF16, (16, 7), 2), (BF16, (2, 3), 3)])
def test_keep_drafted(ops, dtype, shape, axis):
    P, layers = shape[axis - 2], 3
    past, new = [0, 3, 5 * P - 1, 2 * P + 1], [9, 12, 40, 1]
    batch = plain.Batch(past, new, P, "cuda", table_rows=True)
    slab = torch.randint(0, 120, (layers, batch.pages, *shape), generator=torch.Generator().manual_seed(3)).to(dtype)
    paths = [[0, 1, 2, 3, 8], [0, 5, 6, 11], [2, 3, 17, 20, 21, 30, 31, 38, 39], [0]]
    length = max(len(p) for p in paths) + 2
    path = torch.full((4, length), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p)
    path[0, 5] = 8                                            # does not rise: the path ended in front of it
    want = slab.clone().movedim(axis, 2)
    old = want.clone()
    for b, p in enumerate(paths):
        e = batch.entries(b)
        for d, i in enumerate(p):
            to, source = int(e[past[b] + d]), int(e[past[b] + i])
            want[:, to // P, to % P] = old[:, source // P, source % P]
    given = slab.cuda()
    ops.keep_drafted(given, axis, batch.meta.groups[0].block_table, batch.meta.table_rows, batch.meta.kv_len - torch.tensor(new).int().cuda(),
                     path.cuda())
    assert torch.equal(given.cpu().movedim(axis, 2), want)


def test_keep_drafted_stops_at_what_has_no_page(ops):
    slab = torch.arange(1 * 4 * 4 * 2, dtype=torch.float32).view(1, 4, 4, 2).cuda()
    table = torch.tensor([[2, 0, -1], [1, 9, 3]], dtype=torch.int32, device="cuda")        # a page given back, one outside the slab
    past = torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    path = torch.tensor([[1, 2, 7, 8], [0, 2, 3, 4]], dtype=torch.int32, device="cuda")
    want = slab.clone()
    want[0, 2, 2], want[0, 2, 3] = slab[0, 2, 3], slab[0, 0, 0]
    want[0, 1, 2] = slab[0, 1, 3]
    ops.keep_drafted(slab, 2, table, None, past, path)
    assert torch.equal(slab, want)
    ops.keep_drafted(slab, 2, table, None, torch.tensor([-1, 11], dtype=torch.int32, device="cuda"), path)
    assert torch.equal(slab, want)


@pytest.mark.parametrize("path", [[3, 0, 1], [1, 0, 1, 1, 1], [2, -7, -6, -5, -4, -3]])
def test_keep_drafted_at_the_end_of_a_table(ops, path):
    """What stands behind the end of a path names no place, whatever it says: behind the end of the last row there is no table. (The table here is
    the front of a larger tensor.)"""
    P, past = 4, 12
    slab = torch.arange(1 * 8 * P, dtype=torch.float32).view(1, 8, P).cuda()
    held = torch.arange(8, dtype=torch.int32, device="cuda")
    table = held[:4].view(1, 4)
    want = slab.clone()
    before = -1
    for d, i in enumerate(path):
        if i <= before or past + i >= 4 * P:
            break
        want[0, (past + d) // P, (past + d) % P] = slab[0, (past + i) // P, (past + i) % P]
        before = i
    begin = torch.tensor([past], dtype=torch.int32, device="cuda")
    ops.keep_drafted(slab, 2, table, None, begin, torch.tensor([path], dtype=torch.int32, device="cuda"))
    assert torch.equal(slab, want)


@pytest.mark.parametrize("path", [[3, 1], [4, 6, 2], [2, 1, -1], [5, 0, 2], [0, 3, 2, 3], [1, -1, 2, 3, 4], [0, 1, 1, 3], [0, 1, 2, 3], [3, 9, 10, 3, 4, 5]])
def test_keep_drafted_moves_what_stands_in_front_of_a_paths_end(ops, path):
    """Whatever stands behind it: the number of its own place among them."""
    P = 4
    slab = torch.randint(0, 1 << 20, (2, 16, 3, P), dtype=torch.int32, generator=torch.Generator().manual_seed(1))
    past = torch.tensor([0, 5], dtype=torch.int32)
    pages = torch.randperm(16, generator=torch.Generator().manual_seed(2)).int().view(2, 8)
    want = slab.clone()
    for b in range(2):
        before = -1
        for d, i in enumerate(path):
            if i <= before:
                break
            to, source = int(past[b]) + d, int(past[b]) + i
            want[:, pages[b, to // P], :, to % P] = slab[:, pages[b, source // P], :, source % P]
            before = i
    given = slab.cuda()
    ops.keep_drafted(given, 3, pages.cuda(), None, past.cuda(), torch.tensor([path] * 2, dtype=torch.int32, device="cuda"))
    assert torch.equal(given.cpu(), want)


@pytest.mark.parametrize("end", [[], [300, 301], [-1], [550], [551, 551]])
def test_keep_drafted_of_a_path_longer_than_a_block(ops, end):
    """Entries of a path are taken 256 at a time: the first of them stay where they are, the others move, and it ends among the third 256."""
    P = 16
    path = list(range(250)) + list(range(260, 560)) + end
    slab = torch.randint(0, 1 << 20, (1, 40, P), dtype=torch.int32, generator=torch.Generator().manual_seed(1))
    table = torch.randperm(40, generator=torch.Generator().manual_seed(2)).int()[None]
    want, before = slab.clone(), -1
    for d, i in enumerate(path):
        if i <= before:
            break
        want[0, table[0, (7 + d) // P], (7 + d) % P] = slab[0, table[0, (7 + i) // P], (7 + i) % P]
        before = i
    given = slab.cuda()
    ops.keep_drafted(given, 2, table.cuda(), None, torch.tensor([7], dtype=torch.int32, device="cuda"), torch.tensor([path], dtype=torch.int32, device="cuda"))
    assert torch.equal(given.cpu(), want)


# -------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("act, eight", [(BF16, True), (F32, True), (BF16, False), (F32, False)])
def test_a_tree_kept_is_what_its_path_alone_leaves(ops, act, eight):
    """Write, attention of the tree, keep, attention behind it: as if only the accepted tokens had come, one after the other."""
    H, KH, D, P = 12, 2, 128, 16
    past, new = [29, 0], [11, 6]
    batch = tree_batch(past, new, P, seed=11)
    gen = torch.Generator().manual_seed(12)
    qkv = torch.randn(17, (H + 2 * KH) * D, generator=gen).to(act).cuda()
    freq = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().cuda()
    kind = "e4m3" if eight else act
    cache, _, _ = plain.random_cache(batch, KH, D, kind, 13, "cuda", 0.0)
    clone = lambda c: EightBitCache(*(getattr(c, n).clone() for n in ("k", "v", "k_scale", "v_scale"))) if eight else tuple(t.clone() for t in c)
    serial = clone(cache)

    def write(x, meta, c):
        if eight:
            return ops.rope_kv_write_e4m3(x, meta, 0, c, freq, H, KH, D, True)
        return ops.rope_kv_write(x.clone(), meta, 0, *c, freq, H, KH, D, True)

    def attend(q, meta, c):
        if meta.tree is not None:
            return ops.tree_attention(q, meta, 0, c, H, KH, D, D ** -0.5, None)
        if eight:
            return ops.paged_attention_e4m3(q, meta, 0, c, H, KH, D, D ** -0.5, None)
        return ops.paged_attention(q, meta, 0, *c, H, KH, D, D ** -0.5, None)

    of_tree = attend(write(qkv, batch.meta, cache), batch.meta, cache)
    # the deepest token's path of each request
    paths = []
    for b, sees in enumerate(batch.sees):
        deepest = int(sees.sum(1).argmax())
        paths.append(sees[deepest].nonzero()[:, 0].tolist())
    length = max(len(p) for p in paths)
    path = torch.full((2, length), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p)
    held = [(cache.k, 3), (cache.v, 4), (cache.k_scale, 3), (cache.v_scale, 3)] if eight else [(cache[0], 3), (cache[1], 4)]
    begin = torch.tensor(past, dtype=torch.int32, device="cuda")
    for slab, axis in held:
        ops.keep_drafted(slab[None], axis, batch.meta.groups[0].block_table, None, begin, path.cuda())

    # Two kernels with other orders of sums: each is within `attention_bound` of the same value. The sum of a score's products' sizes is at
    # most the product of the norms, a result at most the largest value.
    keys, values = (x.reshape(-1, D) for x in by_slot(cache)[0]) if eight else (
        cache[0].cpu().double().reshape(-1, D), cache[1].cpu().double().transpose(-1, -2).reshape(-1, D))
    heads = qkv[:, :H * D].cpu().double().view(-1, D)               # (a rotation keeps the norm; its rounding is far below the factor 1.1)
    largest = values.abs().max()
    tolerance = 2 * float(plain.attention_bound(largest, largest, 1.1 * heads.norm(dim=1).max() * keys.norm(dim=1).max() * D ** -0.5,
                                                max(past) + max(new), D, act))
    for d in range(length):
        rows = [b for b in range(2) if d < len(paths[b])]
        one = plain.Batch([past[b] + d for b in rows], [1] * len(rows), P, "cuda")
        one.meta.groups[0].block_table = batch.meta.groups[0].block_table[torch.tensor(rows).cuda()].contiguous()
        at = [batch.entries(b)[past[b] + d] for b in rows]
        one.meta.groups[0].slots = torch.tensor(at).int().cuda()
        tokens = torch.tensor([int(batch.cu[b]) + paths[b][d] for b in rows]).cuda()
        q = write(qkv[tokens], one.meta, serial)
        away = (attend(q, one.meta, serial).float() - of_tree[tokens].float()).abs().max()
        assert float(away) < tolerance, (d, float(away))
    for b in range(2):
        slots = batch.entries(b)[:past[b] + len(paths[b])].long().cuda()
        for a, c in zip(*((x.k, x.v, x.k_scale, x.v_scale) if eight else x for x in (cache, serial))):
            axis = 3 if a.shape[2] == D and a.dim() == 4 and a.shape[3] == P else 2
            pick = lambda t: t.view(torch.uint8 if eight else t.dtype).movedim(axis, 1)[slots // P, slots % P]
            assert torch.equal(pick(a), pick(c))


def test_captured_and_replayed_on_another_stream(ops):
    """All operations in one graph: every replay gives what the eager calls give, with eager work between the replays."""
    H, KH, D, P = 12, 2, 128, 16
    single, tree = plain.Batch([900, 3100], [1, 1], P, "cuda"), tree_batch([2000, 700], [300, 30], P, seed=1)
    freq = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().cuda()
    c1, _, _ = plain.random_cache(single, KH, D, "e4m3", 1, "cuda", 0.0)
    c2, _, _ = plain.random_cache(tree, KH, D, BF16, 2, "cuda", 0.0)
    qkv = torch.randn(2, (H + 2 * KH) * D, device="cuda").bfloat16()
    drafted = torch.randn(330, H * D, device="cuda").bfloat16()

    def work():
        q = ops.rope_kv_write_e4m3(qkv, single.meta, 0, c1, freq, H, KH, D, True)
        return (ops.paged_attention_e4m3(q, single.meta, 0, c1, H, KH, D, 0.1, None), *ops.read_kv_e4m3(c1, single.meta.groups[0].slots, BF16),
                ops.tree_attention(drafted, tree.meta, 0, c2, H, KH, D, 0.1, None))

    work()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = work()
    second = torch.cuda.CUDAGraph()                      # of the same step: its parts are its own
    with torch.cuda.graph(second, stream=stream):
        work()
    del second
    # the step's description is made anew: what the graph works in is not the eager calls'
    single.meta.scratch.clear()
    tree.meta.scratch.clear()
    filler = [torch.full((1 << 20,), math.nan, device="cuda") for _ in range(8)]
    for i in range(4):
        qkv.copy_(torch.randn_like(qkv))
        drafted.copy_(torch.randn_like(drafted))
        want = [t.clone() for t in work()]
        for t in out:
            t.fill_(7)
        filler[i].add_(1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("H, KH, D, past, new, other_past, other_new", [
    (28, 4, 128, [4000, 100], [70, 34], [500, 4100], [30, 74]),
    (80, 1, 32, [100, 20], [72, 32], [90, 70], [66, 38]),            # all entries in one walk; a tile more than before
])
def test_a_graph_replayed_with_other_requests(ops, H, KH, D, past, new, other_past, other_new):
    """What the host knows when a graph is captured need not hold when it is replayed: another cut of the same tokens into requests."""
    P = 16
    pages = lambda past, new: max(-(-(p + n) // P) for p, n in zip(past, new))
    first = tree_batch(past, new, P, seed=1, spare=max(1, 1 + pages(other_past, other_new) - pages(past, new)))
    other = tree_batch(other_past, other_new, P, seed=2, spare=max(1, 1 + pages(past, new) - pages(other_past, other_new)))
    cache, _, _ = plain.random_cache(other, KH, D, BF16, 2, "cuda", 0.0)
    q = torch.randn(104, H * D, device="cuda").bfloat16()
    meta = first.meta
    meta.max_q, meta.max_kv = (max(getattr(b.meta, name) for b in (first, other)) for name in ("max_q", "max_kv"))
    run = lambda m: ops.tree_attention(q, m, 0, cache, H, KH, D, 0.1, None)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(meta)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = run(meta)
    for name in ("positions", "token_request", "cu_q", "kv_len", "tree"):
        getattr(meta, name).copy_(getattr(other.meta, name))
    meta.groups[0].block_table.copy_(other.meta.groups[0].block_table)
    # (cut into other walks, so the sums are added up in another order: float32 roundings, and one of the result in bfloat16)
    want = run(other.meta).float()
    for _ in range(3):
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert ((out.float() - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -7).all()
