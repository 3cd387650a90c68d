"""The paged cache's operators restated in 64 bits, row by row, and inputs for them.  Nothing here uses the package."""
import math

import torch

E_MIN, E_MAX = -24, 40


def step_of(top: float) -> float:
    """Smallest 2^e, e in [-24, 40], with top <= 127 * 2^e."""
    for e in range(E_MIN, E_MAX):
        if top <= 127 * 2.0 ** e:
            return 2.0 ** e
    return 2.0 ** E_MAX


def bounds_of(keys):
    """(lowest, highest) [2, dim] as whole numbers, and the step, of keys [n, dim]."""
    keys = keys.double()
    lo, hi = keys.amin(0), keys.amax(0)
    s = step_of(float(torch.maximum(lo.abs(), hi.abs()).max()))
    return torch.stack([torch.floor(lo / s), torch.ceil(hi / s)]).clamp(-127, 127), s


class Setup:
    """A pool with random contents, sequences of given lengths with pages in random order, and new rows."""

    def __init__(self, seed, *, dtype, dim, page, heads, kv_heads, new, lens, prefix=0, tokens_first=False, padding=0, spare=3, leading=0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.dim, self.page, self.heads, self.kv_heads = dtype, dim, page, heads, kv_heads
        self.new, self.lens, self.prefix = list(new), list(lens), prefix
        need = [max(0, -(-n // page)) for n in lens]
        pre = -(-prefix // page)
        self.pages = sum(need) + pre + spare
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max([1] + need)), -1, dtype=torch.int32)
        at = pre
        for b, c in enumerate(need):
            self.table[b, :c] = order[at:at + c]
            at += c
        self.prefix_pages = order[:pre].clone()
        self.offsets = [leading]
        for n in new:
            self.offsets.append(self.offsets[-1] + n)
        self.tokens = self.offsets[-1] + padding
        shape = (self.pages, page, kv_heads, dim) if tokens_first else (self.pages, kv_heads, page, dim)
        k, v = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
        if tokens_first:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        k += torch.randn(self.pages, kv_heads, 1, dim, generator=g).to(dtype)
        self.k, self.v, self.tokens_first = k, v, tokens_first
        self.bounds = torch.zeros(self.pages, kv_heads, 2, dim, dtype=torch.int8)
        self.scales = torch.full((self.pages, kv_heads), 2.0 ** E_MIN)
        for p in range(self.pages):
            for h in range(kv_heads):
                both, s = bounds_of(k[p, h])
                self.bounds[p, h], self.scales[p, h] = both.to(torch.int8), s
        self.q = torch.randn(self.tokens, heads, dim, generator=g).to(dtype)
        self.k_new = torch.randn(self.tokens, kv_heads, dim, generator=g).to(dtype)
        self.v_new = torch.randn(self.tokens, kv_heads, dim, generator=g).to(dtype)

    def rows(self):
        """(row, sequence, position) of every row of a sequence."""
        for b in range(len(self.lens)):
            for j in range(self.new[b]):
                yield self.offsets[b] + j, b, self.lens[b] - self.new[b] + j

    def page_at(self, b, index):
        """Pool page of place `index` of sequence b, or None."""
        if not 0 <= index < self.table.shape[1]:
            return None
        p = int(self.table[b, index])
        return p if 0 <= p < self.pages else None

    def own_keys(self, b, pos, indices=None):
        """(page, place) of the keys that a row at `pos` sees, of all pages or the given ones."""
        out = []
        for i in (range(self.table.shape[1]) if indices is None else indices):
            p = self.page_at(b, i)
            if p is not None:
                out += [(p, o) for o in range(self.page) if i * self.page + o <= pos]
        return out

    def prefix_keys(self):
        out = []
        for i, p in enumerate(self.prefix_pages.tolist()):
            if 0 <= p < self.pages:
                out += [(p, o) for o in range(self.page) if i * self.page + o < self.prefix]
        return out


def attention(s, q_row, h, keys, scale):
    """(out, lse, tolerance of out, tolerance of lse) of one query row over keys [(page, place)] of key head h."""
    if not keys:
        return torch.zeros(s.dim, dtype=torch.float64), -math.inf, torch.full((s.dim,), 0.0, dtype=torch.float64), 0.0
    pp, oo = [a for a, _ in keys], [b for _, b in keys]
    k, v, q = s.k[pp, h, oo].double(), s.v[pp, h, oo].double(), q_row.double()
    logits = k @ q * scale
    lse = torch.logsumexp(logits, 0)
    w = torch.exp(logits - lse)
    out = w @ v
    # a product of `dim` terms in 32 bits is off by at most dim * 2^-23 of the sum of its magnitudes (the matrix unit may cut where
    # it does not round); scaling it and taking it to powers of two add two roundings of its own size; the exponential is
    # off by 2^-22 relative, sums of weights and values by less than that per 64 keys that follow each other
    delta = float((k.abs() @ q.abs()).max()) * scale * (s.dim + 4) * 2.0 ** -23 + 2.0 ** -18
    half = torch.finfo(s.dtype).eps / 2
    mass = w @ v.abs()
    # weights are rounded to the type (half a step each), so is the result
    tol = out.abs() * half + mass * (half + 2 * delta) * (1 + half) + torch.finfo(s.dtype).tiny
    return out, float(lse), tol, delta + abs(float(lse)) * 2.0 ** -22


def attend(s, scale=None):
    """{row: (out [heads, dim], lse [heads], tolerances)} over the prefix and the own keys."""
    scale = s.dim ** -0.5 if scale is None else scale
    group, pre = s.heads // s.kv_heads, s.prefix_keys()
    return {t: [attention(s, s.q[t, j], j // group, pre + s.own_keys(b, p), scale) for j in range(s.heads)] for t, b, p in s.rows()}


def choose(s, t, h, b, pos, budget, first, recent):
    seen = min(pos + 1, s.table.shape[1] * s.page)
    n = max(0, -(-seen // s.page))
    if n <= budget:
        return list(range(n))
    group = s.heads // s.kv_heads
    score = {}
    for i in range(first, n - recent):
        p = s.page_at(b, i)
        best = -math.inf
        if p is not None:
            lo, hi = s.bounds[p, h].double()
            for j in range(h * group, (h + 1) * group):
                q = s.q[t, j].double()
                step = step_of(float(q.abs().max()))
                q8 = torch.round(q / step).clamp(-127, 127)
                best = max(best, float(torch.maximum(q8 * lo, q8 * hi).sum()) * step * float(s.scales[p, h]))
        score[i] = best
    order = sorted(score, key=lambda i: (-score[i], i))[:budget - first - recent]
    return sorted([*range(first), *order, *range(n - recent, n)])


def attend_selected(s, budget, first, recent, scale=None):
    scale = s.dim ** -0.5 if scale is None else scale
    group = s.heads // s.kv_heads
    out, pages = {}, {}
    for t, b, p in s.rows():
        picks = [choose(s, t, h, b, p, budget, first, recent) for h in range(s.kv_heads)]
        pages[t] = picks
        out[t] = [attention(s, s.q[t, j], j // group, s.own_keys(b, min(p, s.table.shape[1] * s.page - 1), picks[j // group]), scale) for j in range(s.heads)]
    return out, pages


def rotate(x, cos, sin, interleaved):
    """x [heads, dim] turned by one position's angles, and the tolerance of 32-bit arithmetic rounded to x's type."""
    half = cos.numel()
    y, mag = x.double().clone(), x.double().abs()
    i1 = torch.arange(half) * 2 if interleaved else torch.arange(half)
    i2 = i1 + 1 if interleaved else i1 + half
    c, s, x1, x2 = cos.double(), sin.double(), x[:, i1].double(), x[:, i2].double()
    y[:, i1], y[:, i2] = x1 * c - x2 * s, x2 * c + x1 * s
    mag = y.abs() * 0
    mag[:, i1] = mag[:, i2] = (x1.abs() + x2.abs())
    # two products and a sum, each half a step of 2^-23 off, then half a step of the type
    return y, y.abs() * torch.finfo(x.dtype).eps / 2 + mag * 2 * 2.0 ** -24 * (1 + torch.finfo(x.dtype).eps) + 2.0 ** -25


def attend_sequence(s, scale=None, weight_step=None, least=0.0, terms=None):
    """attend() for a setup of one sequence, all rows of a head at once: (out [new, heads, dim], lse [new, heads], their tolerances) of the
    sequence's rows in order.  weight_step: half a step of what the weights are rounded to (None: the type's); least:
    half of the smallest step that a weight has, relative to the row's largest; terms: channels of the queries that are not zero (None: all)."""
    assert len(s.lens) == 1
    scale = s.dim ** -0.5 if scale is None else scale
    pre, own = s.prefix_keys(), s.own_keys(0, s.lens[0] - 1)
    pp, oo = [p for p, _ in pre + own], [o for _, o in pre + own]
    place = [i * s.page + o for i in range(s.table.shape[1]) if s.page_at(0, i) is not None for o in range(s.page) if i * s.page + o < s.lens[0]]
    rows = [(t, p) for t, _, p in s.rows()]
    at = [t for t, _ in rows]
    pos = torch.tensor([p for _, p in rows])
    hidden = torch.cat([torch.zeros(len(rows), len(pre), dtype=torch.bool), torch.tensor(place, dtype=torch.long)[None] > pos[:, None]], 1)
    group, half = s.heads // s.kv_heads, torch.finfo(s.dtype).eps / 2
    step = half if weight_step is None else weight_step
    out, lse = torch.zeros(len(rows), s.heads, s.dim, dtype=torch.float64), torch.zeros(len(rows), s.heads, dtype=torch.float64)
    tol, ltol = out.clone(), lse.clone()
    for h in range(s.kv_heads):
        k, v = s.k[pp, h, oo].double(), s.v[pp, h, oo].double()
        for j in range(h * group, (h + 1) * group):
            q = s.q[at, j].double()
            logits = (q @ k.T * scale).masked_fill(hidden, -math.inf)
            lse[:, j] = torch.logsumexp(logits, -1)
            w = torch.exp(logits - lse[:, j, None])
            out[:, j] = w @ v
            # the tolerances of attention() above
            delta = (q.abs() @ k.abs().T).masked_fill(hidden, 0.0).amax(-1) * scale * ((s.dim if terms is None else terms) + 4) * 2.0 ** -23 + 2.0 ** -18
            tol[:, j] = out[:, j].abs() * half + (w @ v.abs()) * (step + 2 * delta)[:, None] * (1 + half) + torch.finfo(s.dtype).tiny * half
            tol[:, j] += least * w.amax(-1, keepdim=True) * ((~hidden).double() @ v.abs())
            ltol[:, j] = delta + lse[:, j].abs() * 2.0 ** -22
    return out, lse, tol, ltol


def prefix_parts(tokens, group, kv_heads, prefix, multiprocessors):
    """What the tensor-memory kernel for a prefix makes of these sizes (kv_prefix_plan of csrc/kv_cache.cuh, restated): whether two tiles of
    rows share a block, and for each group of blocks the (key head, tiles of keys) of its parts."""
    rows = 128 // group * group
    row_tiles = -(-tokens * group // rows)
    paired = row_tiles > 1
    units, tiles = ((row_tiles + 1) // 2 if paired else 1), -(-prefix // 128)
    groups = min(multiprocessors // units if units < multiprocessors else 1, kv_heads * tiles)
    places, per = tiles, -(-kv_heads * tiles // groups)
    of_head = groups // kv_heads
    if of_head > 0 and -(-tiles // of_head) <= per + 4:
        per, groups = -(-tiles // of_head), of_head * kv_heads
        places = of_head * per
    parts = []
    for g in range(groups):
        mine = {}
        for at in range(g * per, min((g + 1) * per, kv_heads * places)):
            if at % places < tiles:
                mine[at // places] = mine.get(at // places, 0) + 1
        parts.append(list(mine.items()))
    return paired, units, parts
