"""What the operations on caches in 8 bits and on drafted tokens refuse, found on the host before anything is launched."""

import pytest
import torch

import plain_cache as plain
from distie_amd.kernels.hip_ops import HipOps, KernelError
from distie_amd.kernels.interface import EightBitCache

H, KH, D, P = 4, 2, 32, 16


class NoLaunch:
    def __getattr__(self, name):
        raise AssertionError(f"{name} would be launched")


@pytest.fixture
def ops():
    """The checks alone: tensors on the CPU, and no library behind them."""
    ops = HipOps.__new__(HipOps)
    ops.device = torch.device("cpu")
    ops._ops = NoLaunch()
    ops._attn = {D: NoLaunch(), 3: NoLaunch()}
    ops._stream = lambda: None
    return ops


def batch(tree=False, **more):
    return plain.Batch([5, 0], [3, 1], P, tree=[torch.ones(3, 3, dtype=torch.bool), torch.ones(1, 1, dtype=torch.bool)] if tree else None, **more)


def cache(pages=4, **changed):
    codes = lambda *shape: torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn)
    held = dict(k=codes(pages, KH, P, D), v=codes(pages, KH, D, P), k_scale=torch.ones(pages, KH, P, dtype=torch.uint8),
                v_scale=torch.ones(pages, KH, P, dtype=torch.uint8))
    held.update(changed)
    return EightBitCache(**held)


QKV = torch.zeros(4, (H + 2 * KH) * D)
BAD_CACHES = [dict(k=torch.zeros(4, KH, P, D, dtype=torch.uint8)), dict(v=torch.zeros(4, KH, D, P)),
              dict(k=torch.zeros(4, KH, D, P, dtype=torch.uint8).view(torch.float8_e4m3fn)),
              dict(v=torch.zeros(3, KH, D, P, dtype=torch.uint8).view(torch.float8_e4m3fn)),
              dict(k_scale=torch.ones(4, KH, P)), dict(v_scale=torch.ones(4, KH, dtype=torch.uint8)),
              dict(k_scale=torch.ones(4, P, KH, dtype=torch.uint8).transpose(1, 2))]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_caches_that_are_not_in_8_bits(ops, bad):
    wrong = cache(**bad)
    with pytest.raises(KernelError):
        ops.rope_kv_write_e4m3(QKV, batch().meta, 0, wrong, None, H, KH, D, True)
    with pytest.raises(KernelError):
        ops.paged_attention_e4m3(QKV, batch().meta, 0, wrong, H, KH, D, 1.0, None)
    with pytest.raises(KernelError):
        ops.tree_attention(QKV, batch(True).meta, 0, wrong, H, KH, D, 1.0, None)
    with pytest.raises(KernelError):
        ops.read_kv_e4m3(wrong, torch.zeros(3, dtype=torch.int32), torch.float32)


def test_write_refuses(ops):
    freq = torch.ones(D // 2)
    call = lambda qkv=QKV, meta=None, freq=freq, heads=H, kv=KH, dim=D, c=None: ops.rope_kv_write_e4m3(
        qkv, meta or batch().meta, 0, c or cache(), freq, heads, kv, dim, True)
    short = batch().meta
    short.groups[0].slots = short.groups[0].slots[:3]
    wide = batch().meta
    wide.groups[0].slots = wide.groups[0].slots.long()
    for bad in (dict(qkv=QKV[:3]), dict(qkv=QKV[:, :-1]), dict(qkv=QKV.T.contiguous().T), dict(qkv=QKV.half()), dict(freq=torch.ones(D)), dict(freq=freq.double()),
                dict(heads=3), dict(kv=0), dict(dim=33), dict(meta=short), dict(meta=wide), dict(c=(1, 2))):
        with pytest.raises(KernelError):
            call(**bad)


def test_read_refuses(ops):
    for slots, dtype in ((torch.zeros(3, dtype=torch.int64), torch.float32), (torch.zeros(1, 3, dtype=torch.int32), torch.float32),
                         (torch.zeros(3, dtype=torch.int32), torch.float16)):
        with pytest.raises(KernelError):
            ops.read_kv_e4m3(cache(), slots, dtype)


def test_attention_refuses(ops):
    call = lambda q=QKV, meta=None, c=None, heads=H, kv=KH, dim=D, scale=1.0, window=None: ops.paged_attention_e4m3(
        q, meta or batch().meta, 0, c or cache(), heads, kv, dim, scale, window)
    rows = batch(table_rows=True).meta
    rows.table_rows = rows.table_rows[:1]
    long = batch().meta
    long.kv_len = long.kv_len.long()
    table = batch().meta
    table.groups[0].block_table = table.groups[0].block_table[:1]
    for bad in (dict(q=QKV[:3]), dict(q=QKV[:, :H * D - 1]), dict(q=QKV.half()), dict(q=QKV.T.contiguous().T), dict(heads=3), dict(kv=0), dict(dim=31), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("nan")), dict(window=0), dict(window=-2), dict(meta=batch(True).meta), dict(meta=rows),
                dict(meta=long), dict(meta=table), dict(c=(torch.zeros(4, KH, P, D), torch.zeros(4, KH, D, P)))):
        with pytest.raises(KernelError):
            call(**bad)


def test_attention_over_a_plain_cache_refuses_trees(ops):
    """By positions alone it would let a drafted token see its siblings."""
    with pytest.raises(KernelError, match="tree_attention"):
        ops.paged_attention(QKV, batch(True).meta, 0, torch.zeros(4, KH, P, D), torch.zeros(4, KH, D, P), H, KH, D, 1.0, None)


def test_trees_refuse(ops):
    plain_cache = torch.zeros(4, KH, P, D), torch.zeros(4, KH, D, P)
    call = lambda meta, c=plain_cache: ops.tree_attention(QKV, meta, 0, c, H, KH, D, 1.0, None)
    wrong = [batch(True).meta for _ in range(3)]
    wrong[0].tree = wrong[0].tree.int()
    wrong[1].tree = wrong[1].tree[:3]
    wrong[2].max_q = 65
    for meta in [batch().meta] + wrong:
        with pytest.raises(KernelError):
            call(meta)
    for bad in ((plain_cache[0].bfloat16(), plain_cache[1].bfloat16()), (plain_cache[0], plain_cache[1].bfloat16()), (plain_cache[1], plain_cache[0]),
                (plain_cache[0].half(), plain_cache[1].half())):
        with pytest.raises(KernelError):
            call(batch(True).meta, bad)


def test_keep_refuses(ops):
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    slab = torch.zeros(2, 4, KH, P, D)
    good = dict(slab=slab, page_axis=3, table=ints(2, 3), table_rows=None, past=ints(2), path=ints(2, 5))
    for bad in (dict(page_axis=1), dict(page_axis=5), dict(slab=slab.transpose(0, 1)), dict(table=ints(3, 3)), dict(table=ints(3)), dict(table=ints(2, 3).long()),
                dict(past=ints(3)), dict(past=ints(2, 1)), dict(path=ints(5)), dict(path=ints(2, 5).long()), dict(table_rows=ints(3)), dict(slab=slab[0, 0])):
        with pytest.raises(KernelError):
            ops.keep_drafted(**{**good, **bad})
    ops.keep_drafted(**{**good, "path": ints(2, 0)})            # nothing to do, nothing launched


class Launches:
    """In place of a head size's library: what it would have launched, with a tensor's shape for a tensor."""

    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        shown = lambda a: tuple(a.shape) if isinstance(a, torch.Tensor) else a
        return lambda *a: self.made.append((name, *(shown(x) for x in a))) or 0


def plan_of(ops, act, meta, tree, heads=(28, 4, 128)):
    """The launches of one call, and the rows and requests that their parts hold."""
    H, KH, D = heads
    ops._attn[D] = lib = Launches()
    lib.distie_cache_attention_shares = lambda: 64
    pages = 4
    codes = lambda *shape: torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn)
    held = EightBitCache(codes(pages, KH, P, D), codes(pages, KH, D, P), *(torch.ones(pages, KH, P, dtype=torch.uint8) for _ in range(2)))
    call = ops.tree_attention if tree else ops.paged_attention_e4m3
    call(torch.zeros(meta.num_tokens, H * D, dtype=act), meta, 0, held, H, KH, D, 1.0, None)
    return [(name, *(x for x in a[1:] if not isinstance(x, int) or x < 1 << 40)) for name, *a in lib.made]          # (without q's address)


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("change", ["most", "contexts", "contexts in place", "requests", "tokens", "captured"])
def test_a_description_that_changes_gets_launches_of_its_own(ops, monkeypatch, act, tree, change):
    """What a step's launches are made by is looked at in every call: more tokens a request than before, longer contexts under the same bound,
    more requests or tokens need more workgroups and longer parts than the call before had."""
    monkeypatch.setattr(ops, "_empty", lambda shape, dtype: torch.empty(shape, dtype=dtype), raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    def step(past, new, known):
        trees = [torch.ones(n, n, dtype=torch.bool).tril() for n in new] if tree else None
        meta = plain.Batch(past, new, P, tree=trees).meta
        meta.groups[0].block_table = torch.zeros(meta.num_requests, 600, dtype=torch.int32)
        meta.max_kv, meta.all_decode = 700 if change == "captured" else 9000, False
        if not known:
            meta.host_cu_q = meta.host_past = None
        return meta

    known = change.startswith("contexts")
    before, after = {"most": (([8, 40], [3, 4]), ([8, 40], [3, 200])), "requests": (([100], [30]), ([100, 40, 8000], [3, 26, 1])),
                     "tokens": (([100, 40], [30, 20]), ([100, 40], [30, 30])), "captured": (([100, 40], [1, 1]), ([100, 40], [1, 1]))}.get(
                         change, (([100, 40], [3, 200]), ([8500, 8000], [3, 200])))
    meta, then = step(*before, known), step(*after, known)
    if change == "tokens":
        meta.max_q = then.max_q = 50
    plan_of(ops, act, meta, tree)
    if change == "contexts in place":
        meta.host_past[:] = then.host_past
        meta.kv_len.copy_(then.kv_len)
    else:
        scratch, cu_q = meta.scratch, meta.host_cu_q
        meta.__dict__.update(then.__dict__)
        meta.scratch, meta.host_cu_q = scratch, cu_q           # (the same array, or none)
    then.scratch = {}
    ops.captured = change == "captured"
    assert plan_of(ops, act, meta, tree) == plan_of(ops, act, then, tree)
