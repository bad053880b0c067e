"""Plain forms, in 64 bits, of a cache in 8 bits and of attention over paged caches, and batches made by hand for them.

Nothing here is shared with the package: codes and powers are found by comparing with every code there is, and attention loops
over the tokens."""

import math

import torch

from distie_amd.kernels.interface import BatchMeta, EightBitCache, GroupMeta

# the 127 sizes that an e4m3 code stands for: 0, 2^-9 .. 448
SIZES = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119],
                     dtype=torch.float64)


def power_of(row):
    """The byte of a row of float64 values."""
    finite = row[torch.isfinite(row)].abs()
    largest = float(finite.max()) if finite.numel() else 0.0
    e = -126
    while e < 127 and largest > 448 * 2.0 ** e:
        e += 1
    return e + 127


def codes_of(row, byte):
    """What the codes of a row stand for, in units of its power: the nearest size, of two equally near the even one."""
    y = row / 2.0 ** (byte - 127)
    away = (y.abs()[:, None] - SIZES).abs()
    nearest = away.argmin(-1)
    tie = (nearest + 1 < 127) & (away.gather(1, (nearest + 1).clamp(max=126)[:, None])[:, 0] == away.gather(1, nearest[:, None])[:, 0])
    nearest = torch.where(tie & (nearest % 2 == 1), nearest + 1, nearest)
    out = torch.copysign(SIZES[nearest], y)
    return torch.where(torch.isfinite(row), out, torch.nan)


def quantised(rows):
    """rows float64 [..., D] -> (values that the codes stand for times their power, bytes)"""
    flat = rows.reshape(-1, rows.shape[-1])
    bytes_ = torch.tensor([power_of(r) for r in flat])
    values = torch.stack([codes_of(r, int(b)) * 2.0 ** (int(b) - 127) for r, b in zip(flat, bytes_)])
    return values.view(rows.shape), bytes_.view(rows.shape[:-1])


def rotated(x, positions, inv_freq):
    """x float64 [T, heads, D], the first 2 len(inv_freq) dimensions of every head turned."""
    pairs = inv_freq.shape[0]
    angle = (positions.double()[:, None] * inv_freq.double())[:, None]
    a, b = x[..., :pairs], x[..., pairs:2 * pairs]
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., 2 * pairs:]], -1)


class Batch:
    """Requests with `past` cached entries and `new` tokens each, on pages given out in a shuffled order; `spare` table entries
    behind every request's pages and the pages that a window has passed are -1."""

    def __init__(self, past, new, page, device="cpu", seed=0, tree=None, positions=None, window=None, table_rows=False, spare=1):
        gen = torch.Generator().manual_seed(seed)
        self.past, self.new, self.page = list(past), list(new), page
        B, T = len(past), sum(new)
        counts = [-(-(p + n) // page) for p, n in zip(past, new)]
        order = torch.randperm(sum(counts) + 1, generator=gen, dtype=torch.int32)
        self.pages = sum(counts) + 1                     # one that no request has
        rows = B + 2 if table_rows else B
        table = torch.full((rows, max(counts) + spare), -1, dtype=torch.int32)
        self.row = torch.randperm(rows, generator=gen)[:B].int() if table_rows else torch.arange(B, dtype=torch.int32)
        at, self.slots = 0, []
        for b, count in enumerate(counts):
            pages = order[at:at + count]
            at += count
            table[self.row[b], :count] = pages
            index = torch.arange(past[b], past[b] + new[b])
            self.slots.append(pages[index // page].long() * page + index % page)
            if window is not None:
                first = max(0, past[b] - window + 1) // page
                table[self.row[b], :first] = -1
        self.slots = torch.cat(self.slots).int() if T else torch.zeros(0, dtype=torch.int32)
        self.table = table
        self.request = torch.repeat_interleave(torch.arange(B), torch.tensor(new)).int()
        self.cu = torch.cat([torch.zeros(1, dtype=torch.long), torch.tensor(new).cumsum(0)])
        self.positions = positions if positions is not None else torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).int()
        self.sees = tree                                  # per request: bool [n, n]
        words = None
        if tree is not None:
            W = -(-max(new) // 64)
            words = torch.zeros(T, W, dtype=torch.int64)
            for b, s in enumerate(tree):
                bits = torch.nn.functional.pad(s, (0, 64 * W - new[b])).view(new[b], W, 64).long()
                words[self.cu[b]:self.cu[b + 1]] = (bits << torch.arange(64)).sum(-1)
        to = lambda t, dtype=torch.int32: None if t is None else t.to(device=device, dtype=dtype)
        self.meta = BatchMeta(
            num_tokens=T, num_requests=B, positions=to(self.positions), token_request=to(self.request), cu_q=to(self.cu),
            kv_len=to(torch.tensor(past) + torch.tensor(new)), state_slots=to(self.row), max_q=max(new), max_kv=max(p + n for p, n in zip(past, new)),
            block_size=page, groups=[GroupMeta(to(table), to(self.slots))], host_cu_q=self.cu.numpy(), host_past=torch.tensor(past).numpy(),
            all_decode=max(new) == 1, table_rows=to(self.row) if table_rows else None, tree=to(words, torch.int64))

    def entries(self, b):
        """Slots of the request's cached entries and of its new ones, in their order (-1: its page was given back)."""
        index = torch.arange(self.past[b] + self.new[b])
        pages = self.table[self.row[b], index // self.page].long()
        return torch.where(pages < 0, -1, pages * self.page + index % self.page)

    def seen_by(self, t, window):
        """bool over the request's entries"""
        b = int(self.request[t])
        past, n, begin, pos = self.past[b], self.new[b], int(self.cu[b]), int(self.positions[t])
        where = torch.arange(past + n)
        if self.sees is None:
            seen = where <= pos
        else:
            seen = torch.cat([torch.ones(past, dtype=torch.bool), self.sees[b][t - begin]])
            where[past:] = self.positions[begin:begin + n].long()
        return seen & (pos - where < window) if window is not None else seen


def attended(q, batch, keys, values, kv_heads, scale, window=None):
    """q float64 [T, H, D]; keys, values float64 [pages * P, KH, D] by slot -> (out float64 [T, H, D], zeros where nothing is seen;
    the same with the values' sizes; the largest sum of |q_d k_d| * scale of a token and head [T, H, 1]; the most keys a token sees)"""
    T, H, D = q.shape
    out, sizes, scores, most = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, 1, dtype=torch.float64), 0
    for t in range(T):
        slots = batch.entries(int(batch.request[t]))
        seen = slots[batch.seen_by(t, window)]
        if not len(seen):
            continue
        assert (seen >= 0).all()
        k, v = keys[seen].transpose(0, 1), values[seen].transpose(0, 1)               # [KH, n, D]
        one = q[t].view(kv_heads, -1, D)
        w = torch.softmax(one @ k.transpose(1, 2) * scale, -1)
        out[t], sizes[t] = (w @ v).view(H, D), (w @ v.abs()).view(H, D)
        scores[t] = (one.abs() @ k.abs().transpose(1, 2)).amax(-1).view(H, 1) * scale
        most = max(most, len(seen))
    return out, sizes, scores, most


def attention_bound(out, sizes, scores, most, dim, act):
    """How far a result may be from `out`. In float32 a score is off by at most (dim + 4) roundings of the sum of its products'
    sizes (the sum itself, the factor, the reference, the exponential), a weight by that relative to itself, numerator and denominator
    alike, and sums of `most` terms by as many roundings of the sum of their sizes. In bfloat16 every weight is rounded once more on
    its way into the product (2^-8 of itself), and the result once."""
    bound = sizes * (2 * (dim + 4) * 2.0 ** -24 * scores + 2 * (most + 8) * 2.0 ** -24)
    if act == torch.bfloat16:
        bound = bound + sizes * 2.0 ** -8
        bound = bound + (out.abs() + bound) * 2.0 ** -8
    return bound + 1e-30


def random_cache(batch, kv_heads, dim, kind, seed, device, garbage=math.nan):
    """-> (cache as the kernels take it, keys, values float64 [pages * P, KH, D] as it holds them). What no request has written
    is `garbage`."""
    gen = torch.Generator().manual_seed(seed)
    P, N = batch.page, batch.pages
    used = torch.zeros(N * P, dtype=torch.bool)
    for b in range(len(batch.past)):
        e = batch.entries(b)
        used[e[e >= 0]] = True
    k, v = (torch.randn(N * P, kv_heads, dim, generator=gen) * torch.exp(torch.randn(N * P, kv_heads, 1, generator=gen) / 2) for _ in range(2))
    k[:, :, 1::17] *= 3
    v += 0.3
    k[~used], v[~used] = garbage, garbage
    by_page = lambda x: x.view(N, P, kv_heads, -1).transpose(1, 2)
    if kind == "e4m3":
        both, held = [], []
        for x in (k, v):
            bits = torch.where(x.isfinite(), x.abs(), 0).amax(-1).view(torch.int32)
            power = ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000)).clamp(-126, 127)
            codes = torch.ldexp(x, -power[..., None]).to(torch.float8_e4m3fn)
            held.append(torch.ldexp(codes.double(), power[..., None]))
            both.append((codes, (power + 127).to(torch.uint8)))
        (kc, kp), (vc, vp) = both
        put = lambda c: by_page(c.view(torch.uint8)).contiguous()
        cache = EightBitCache(put(kc).view(torch.float8_e4m3fn).to(device), put(vc).transpose(-1, -2).contiguous().view(torch.float8_e4m3fn).to(device),
                              by_page(kp[..., None])[..., 0].contiguous().to(device), by_page(vp[..., None])[..., 0].contiguous().to(device))
        return cache, held[0], held[1]
    k, v = k.to(kind), v.to(kind)
    return (by_page(k).contiguous().to(device), by_page(v).transpose(-1, -2).contiguous().to(device)), k.double(), v.double()


def random_tree(n, gen, chain=0.5):
    """bool [n, n]: token 0 is the root, every other one hangs on an earlier one and sees its ancestors and itself -> (sees, depths)"""
    sees, depth = torch.eye(n, dtype=torch.bool), torch.zeros(n, dtype=torch.long)
    for i in range(1, n):
        parent = i - 1 if float(torch.rand((), generator=gen)) < chain else int(torch.randint(i, (), generator=gen))
        sees[i] |= sees[parent]
        depth[i] = depth[parent] + 1
    return sees, depth
