"""GPU: the operators over a caller's paged K/V cache against their formulas in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24          # half a step of fp32, relative
U16 = 2.0 ** -8         # of bf16
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float32)


@pytest.fixture(scope="module")
def api(built_lib):
    from mini_llm_cuda_b200 import api as _api
    return _api


@pytest.fixture(scope="module")
def ops(api):
    return api.Ops(0)


def to_fp4(x, pool_scale):
    """numpy fp32 [..., D] -> codes, e4m3 bytes, as the operator's documentation has it."""
    import torch
    b = x.astype(np.float32).reshape(-1, 16)
    top = np.abs(b).max(-1)
    ratio = np.minimum(top / (np.float32(6) * np.float32(pool_scale)), np.float32(448))
    scale = torch.from_numpy(ratio.astype(np.float32)).to(torch.float8_e4m3fn)
    unit = scale.float().numpy() * np.float32(pool_scale)
    inv = np.where(unit > 0, np.float32(1) / np.where(unit > 0, unit, np.float32(1)), np.float32(0)).astype(np.float32)
    y = b * inv[:, None]
    a = np.minimum(np.abs(y), np.float32(6))
    lo = np.searchsorted(E2M1, a, side="right") - 1
    hi = np.minimum(lo + 1, 7)
    mid = (E2M1[lo] + E2M1[hi]) / 2
    code = np.where((a > mid) | ((a == mid) & (lo % 2 == 1)), hi, lo).astype(np.uint8) | (np.signbit(y).astype(np.uint8) << 3)
    code = code.reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.view(torch.uint8).numpy().reshape(*x.shape[:-1], -1)


def from_fp4(codes, scales, pool_scale):
    """codes, e4m3 bytes (torch) -> values in 64 bits."""
    import torch
    v = torch.tensor(np.concatenate([E2M1, -E2M1]), dtype=torch.float64, device=codes.device)
    c = codes.long()
    x = torch.stack([v[c & 15], v[c >> 4]], dim=-1).flatten(-2)
    s = scales.view(torch.float8_e4m3fn).double().repeat_interleave(16, dim=-1)
    return x * s * float(np.float32(pool_scale))


class Case:
    """A cache with random contents, its sequences' pages anywhere in it, and new rows."""

    def __init__(self, api, new, lens, heads, kv_heads, hd, cache="bf16", rows="bf16", seed=0, ragged=True, extra_rows=0, k_scale=0.02, v_scale=0.01,
                 pages=None, loud=1.0):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        dev = dict(device="cuda")
        self.api, self.new, self.lens, self.heads, self.kv_heads, self.hd, self.cache = api, list(new), list(lens), heads, kv_heads, hd, cache
        self.dt = {"f32": torch.float32, "bf16": torch.bfloat16}[rows]
        need = [max(0, (n + 15) // 16) for n in lens]
        self.n_pages = pages or sum(need) + 3
        perm = torch.randperm(self.n_pages, generator=g, **dev).int()
        self.table = torch.full((len(need), max(need + [1])), -7, dtype=torch.int32, **dev)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        shape = (self.n_pages, kv_heads, 16, hd)
        self.k_scale, self.v_scale, self.kscale, self.vscale = 1.0, 1.0, None, None
        if cache == "fp4":
            self.k_scale, self.v_scale = k_scale, v_scale
            self.kpool, self.vpool = (torch.randint(0, 256, (*shape[:3], hd // 2), dtype=torch.uint8, generator=g, **dev) for _ in range(2))
            self.kscale, self.vscale = ((torch.rand((*shape[:3], hd // 16), generator=g, **dev) * 30 + 1).to(torch.float8_e4m3fn) for _ in range(2))
        else:
            t = {"f32": torch.float32, "bf16": torch.bfloat16}[cache]
            self.kpool, self.vpool = ((torch.randn(shape, generator=g, **dev) * loud).to(t) for _ in range(2))
        self.rows = sum(new) + extra_rows
        self.row_start = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, **dev) if ragged else None
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, **dev)
        randn = lambda w: torch.randn(self.rows, w, generator=g, **dev).to(self.dt)  # noqa: E731
        self.q, self.k, self.v = randn(heads * hd), randn(kv_heads * hd), randn(kv_heads * hd)
        self.describe()

    def describe(self, max_rows=0):
        self.kv = self.api.PagedKV(self.kpool, self.vpool, self.table, kscale=self.kscale, vscale=self.vscale, k_scale=self.k_scale, v_scale=self.v_scale)
        self.nr = self.api.NewRows(self.kv_lens, self.rows, row_start=self.row_start, max_rows=max_rows)

    def cached(self, which, b, length):
        """[kv_heads][length][hd] in 64 bits."""
        ids = self.table[b, :(length + 15) // 16].long()
        pool = getattr(self, which + "pool")[ids]
        x = from_fp4(pool, getattr(self, which + "scale")[ids], getattr(self, which + "_scale")) if self.cache == "fp4" else pool.double()
        return x.permute(1, 0, 2, 3).reshape(self.kv_heads, -1, self.hd)[:, :length]

    def attention(self, window=0, sinks=0, scale=0.0, gate=None, q=None):
        """(answer in 64 bits, bound of the error) of every row that belongs to a sequence; NaN elsewhere."""
        import torch
        q = self.q if q is None else q
        H, D, G = self.heads, self.hd, self.heads // self.kv_heads
        out = torch.full((self.rows, H * D), float("nan"), dtype=torch.float64, device="cuda")
        tol = out.clone()
        scale = scale or 1 / math.sqrt(D)
        r0 = 0
        for b, (n, L) in enumerate(zip(self.new, self.lens)):
            if n == 0:
                continue
            L = max(L, 0)
            p = torch.arange(L - n, L, device="cuda")
            j = torch.arange(L, device="cuda")
            sees = j[None] <= p[:, None]
            if window:
                sees &= (j[None] > p[:, None] - window) | (j[None] < sinks)
            K, V = self.cached("k", b, L), self.cached("v", b, L)
            K, V = torch.nan_to_num(K, 0, 0, 0), torch.nan_to_num(V, 0, 0, 0)      # (a test that plants them hides them from every row)
            qq = q[r0:r0 + n].double().reshape(n, self.kv_heads, G, D).permute(1, 2, 0, 3)
            s = (qq @ K[:, None].transpose(-1, -2) * scale).masked_fill(~sees, -math.inf)
            w = torch.softmax(s, dim=-1).nan_to_num(0)
            o = w @ V[:, None]
            # A score is off by its D products and sums, a weight by twice the largest of these and by the exponential's few steps (the argument
            # is rounded once, relative to a score of up to `most`), a sum over L weights by L steps; matrix cores may cut off where they add, a
            # whole step and not half of one. bf16 rows: probabilities and the result are rounded to bf16, half a step each.
            if L:
                most = (qq.abs() @ K[:, None].abs().transpose(-1, -2) * scale).masked_fill(~sees, 0).amax(-1, keepdim=True)
                big = (w > 0).to(torch.float64) @ V[:, None].abs() * 0 + V.abs().amax((1, 2))[:, None, None, None]
                t = big * U * 2 * (2 * (D + 8) * most + L + 40)
                if self.dt == torch.bfloat16:
                    t = t + 1.1 * U16 * (o.abs() + (w @ V[:, None].abs()))
            else:
                t = torch.zeros_like(o)
            lay = lambda x: x.permute(2, 0, 1, 3).reshape(n, H * D)  # noqa: E731
            out[r0:r0 + n], tol[r0:r0 + n] = lay(o), lay(t)
            r0 += n
        if gate is not None:
            out, tol = out * gate.double(), tol * gate.double() + out.abs() * gate.double() * 2 * U
        return out, tol


def attend(ops, c, window=0, sinks=0, q=None, out=None, **kw):
    import torch
    q = c.q if q is None else q
    if out is None:
        out = torch.full((c.rows, c.heads * c.hd), 777.0, dtype=c.dt, device="cuda")
    ops.attn_paged(c.kv, c.nr, q, out, heads=c.heads, window=window, sinks=sinks, **kw)
    return out


def check(out, want, tol):
    import torch
    used = ~torch.isnan(want)
    assert bool((out[~used] == 777.0).all())
    got = out.double()
    assert bool(torch.isfinite(got[used]).all())
    over = ((got - want).abs() - tol)[used]
    assert float(over.max()) <= 0, f"{float((got - want).abs()[used].max()):.3g} off, {float(over.max()):.3g} over the bound, at {int((over > 0).sum())} places"


TYPES = [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("fp4", "f32"), ("fp4", "bf16"), ("f32", "bf16")]
EDGES = [1, 2, 15, 16, 17, 31, 33, 64, 100, 129, 257, 700]


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 8, 64), (16, 4, 128), (7, 1, 64), (8, 1, 128), (6, 2, 128), (10, 2, 64), (3, 1, 128), (4, 2, 64)])
def test_steps(api, ops, cache, rows, heads, kv_heads, hd):
    """One new token per sequence, contexts at the edges of pages; with and without a window."""
    c = Case(api, [1] * len(EDGES), EDGES, heads, kv_heads, hd, cache, rows, ragged=False, extra_rows=2)
    for window, sinks in ((0, 0), (1, 0), (1, 3), (16, 0), (33, 5), (100, 40), (5000, 4)):
        check(attend(ops, c, window, sinks), *c.attention(window, sinks))
    ops.status()


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 8, 64), (16, 4, 128), (7, 1, 64), (8, 1, 128), (6, 2, 128)])
def test_ragged_rows(api, ops, cache, rows, heads, kv_heads, hd):
    """Prompts, chunks of prompts and single tokens in one call, empty sequences among them, rows behind the last one."""
    new = [1, 0, 5, 17, 2, 130, 1, 0, 64, 3, 300, 33]
    lens = [1, 9, 5, 40, 300, 130, 77, 0, 64, 18, 411, 33]
    c = Case(api, new, lens, heads, kv_heads, hd, cache, rows, extra_rows=3)
    for window, sinks in ((0, 0), (1, 0), (50, 4), (129, 33)):
        check(attend(ops, c, window, sinks), *c.attention(window, sinks))
    ops.status()


@pytest.mark.parametrize("cache,rows", TYPES)
def test_one_long_sequence(api, ops, cache, rows):
    """Splits along the positions: one row, then a few rows of a sequence, far into a context."""
    for new, length in ((1, 5003), (1, 4096), (3, 5003), (4, 2500)):
        c = Case(api, [new], [length], 16, 4, 128, cache, rows)
        for window, sinks in ((0, 0), (3000, 20)):
            check(attend(ops, c, window, sinks), *c.attention(window, sinks))
    ops.status()


@pytest.mark.parametrize("cache,rows", TYPES)
def test_many_sequences(api, ops, cache, rows):
    rng = np.random.default_rng(5)
    lens = rng.integers(1, 400, size=203).tolist()
    c = Case(api, [1] * 203, lens, 16, 8, 64, cache, rows, ragged=False)
    for window, sinks in ((0, 0), (64, 4)):
        check(attend(ops, c, window, sinks), *c.attention(window, sinks))
    new = rng.integers(0, 5, size=203).tolist()
    c = Case(api, new, [n + l for n, l in zip(new, lens)], 16, 8, 64, cache, rows)
    check(attend(ops, c, 64, 4), *c.attention(64, 4))
    ops.status()


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("new", [1, 4, 70])
def test_nothing_visible_and_padding(api, ops, cache, rows, new):
    """Sequences shorter than the rows they bring: rows before position 0 are zeros; the page table of an empty sequence is not read."""
    lens = [0, 0, max(0, new - 1), max(0, new - 3), new, 0]
    c = Case(api, [new] * 6, lens, 4, 2, 64, cache, rows)
    want, tol = c.attention(9, 1)
    out = attend(ops, c, 9, 1)
    check(out, want, tol)
    assert bool((out[:new] == 0).all())
    ops.status()


@pytest.mark.parametrize("cache,rows", [t for t in TYPES if t[0] != "fp4"])
@pytest.mark.parametrize("new", [1, 3, 90])
def test_hidden_positions_hold_no_numbers(api, ops, cache, rows, new):
    """Infinities and NaN at positions that no row sees: behind the last one, between the first ones and the window, in other pages."""
    import torch
    lens = [new + 200, new + 37, new, new + 129]
    window, sinks = 20, 5
    c = Case(api, [new] * 4, lens, 8, 2, 128, cache, rows)
    want, tol = c.attention(window, sinks)
    flat = torch.ones(c.n_pages, 16, dtype=torch.bool, device="cuda")
    for b, L in enumerate(lens):
        for j in range(L):
            if j < sinks or j > L - new - window:
                flat[int(c.table[b, j // 16]), j % 16] = False
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda")
    n = 0
    for pool in (c.kpool, c.vpool):
        v = pool.permute(0, 2, 1, 3)
        v[flat] = bad[(torch.arange(int(flat.sum()), device="cuda") + n) % 3].to(pool.dtype)[:, None, None].expand(-1, c.kv_heads, c.hd)
        n += 1
    check(attend(ops, c, window, sinks), want, tol)


@pytest.mark.parametrize("cache,rows", [t for t in TYPES if t[0] != "fp4"])
@pytest.mark.parametrize("heads,hd", [(2, 64), (8, 128)])
def test_a_later_row_sees_no_number(api, ops, cache, rows, heads, hd):
    """A position that some rows of a sequence see and others do not holds infinities: those that do not see it are as without it, those that
    do get what the formula gives."""
    import torch
    new, L = 40, 60
    c = Case(api, [new], [L], heads, 2, hd, cache, rows)
    want, tol = c.attention()
    at = 45
    page, slot = int(c.table[0, at // 16]), at % 16
    c.vpool[page, :, slot] = math.inf
    out = attend(ops, c)
    before = at - (L - new)                       # rows in front of the position
    got = out.double()
    assert float(((got - want).abs() - tol)[:before].max()) <= 0
    assert bool((got[before:] == math.inf).all())
    c.kpool[page, :, slot] = math.nan
    got = attend(ops, c).double()
    assert float(((got - want).abs() - tol)[:before].max()) <= 0
    assert bool(torch.isnan(got[before:]).all())


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("new", [1, 150])
def test_large_scores(api, ops, cache, rows, new):
    """Scores of some thousands: one position takes all the weight; and all scores equal."""
    import torch
    c = Case(api, [new], [new + 300], 8, 2, 64, cache, rows)
    c.q = (c.q.float() * 300).to(c.dt)
    want, _ = c.attention()
    out = attend(ops, c).double()
    assert bool(torch.isfinite(out).all())
    # a score of up to 300 * 64 * 9 / 8 is off by fp32 roundings of its sum: weights may differ by some percent where two are near
    assert float((out - want).abs().max()) <= 0.1 * float(want.abs().max())
    c.q.zero_()
    check(attend(ops, c), *c.attention())


@pytest.mark.parametrize("cache,rows", [("bf16", "bf16"), ("bf16", "f32"), ("fp4", "bf16")])
@pytest.mark.parametrize("new", [1, 4, 140])
def test_strides_gate_and_scale(api, ops, cache, rows, new):
    """q, out with rows apart, on odd boundaries; gates; a scale of the caller's."""
    import torch
    c = Case(api, [new, new, new], [new + 5, new, new + 130], 8, 2, 64, cache, rows)
    w = c.heads * c.hd
    gate = torch.rand(c.rows, w, device="cuda")
    want, tol = c.attention(50, 2, scale=0.3, gate=gate)
    for off, pad in ((0, 0), (1, 3), (3, 5), (8, 16)):
        qb = torch.zeros(c.rows * (w + pad) + off, dtype=c.dt, device="cuda")
        ob = torch.full((c.rows * (w + pad) + off,), 777.0, dtype=c.dt, device="cuda")
        q, o = (x[off:].as_strided((c.rows, w), (w + pad, 1)) for x in (qb, ob))
        q.copy_(c.q)
        attend(ops, c, 50, 2, q=q, out=o, scale=0.3, gate=gate)
        check(o, want, tol)
        if pad:
            assert bool((ob[off:].as_strided((c.rows - 1, pad), (w + pad, 1), off + w) == 777.0).all())
        assert bool((ob[:off] == 777.0).all())


@pytest.mark.parametrize("cache,rows", TYPES)
def test_same_bits_twice(api, ops, cache, rows):
    c = Case(api, [1, 7, 150, 1], [3000, 900, 700, 40], 16, 4, 128, cache, rows)
    a, b = attend(ops, c, 500, 4), attend(ops, c, 500, 4)
    assert bool((a == b).all())


# ---- append and read -------------------------------------------------------------------------------------------------
def rope_table(length, hd):
    import torch
    inv = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    ang = torch.arange(length, dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], dim=-1).reshape(length, hd).float().cuda()


def rotated(x, cs, heads):
    """fp32 [rows][heads][hd], every product and sum rounded once, as numpy has it."""
    x = x.float().cpu().numpy().reshape(x.shape[0], heads, -1)
    if cs is None:
        return x
    c, s = cs[:, None, 0::2], cs[:, None, 1::2]
    a, b = x[..., 0::2], x[..., 1::2]
    return np.stack([c * a - s * b, s * a + c * b], axis=-1).reshape(x.shape)


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 8, 64), (16, 4, 128), (3, 1, 64)])
@pytest.mark.parametrize("kind", ["steps", "ragged"])
def test_append(api, ops, cache, rows, heads, kv_heads, hd, kind):
    """Every stored row is the rotated one, rounded once; everything else in the pools and in q_out stays; kv_read returns what is stored."""
    import torch
    if kind == "steps":
        new, lens = [1] * 9, [1, 16, 17, 400, 0, 33, 5, 2, 64]
    else:
        new, lens = [1, 0, 40, 17, 3, 5], [9, 4, 40, 100, 1, 70]          # the fifth: two rows of padding
    c = Case(api, new, lens, heads, kv_heads, hd, cache, rows, ragged=kind == "ragged", extra_rows=2)
    c.k[0].zero_()
    c.v[-1].zero_()
    c.k[1] *= 1000
    rope = rope_table(max(lens), hd)
    names = ["kpool", "vpool"] + (["kscale", "vscale"] if cache == "fp4" else [])
    raw = lambda t: t.view(torch.uint8).clone()  # noqa: E731
    want = {n: raw(getattr(c, n)) for n in names}
    q_want = torch.full_like(c.q, 777.0)
    t = 0
    stored = []
    for b, (n, L) in enumerate(zip(new, lens)):
        for i in range(n):
            pos = L - n + i
            if pos >= 0:
                stored.append((t, b, pos))
            t += 1
    ts = [x[0] for x in stored]
    cs = rope.cpu().numpy()[[x[2] for x in stored]]
    kr, vr = rotated(c.k[ts], cs, kv_heads), rotated(c.v[ts], None, kv_heads)
    q_want[ts] = torch.from_numpy(rotated(c.q[ts], cs, heads)).to(c.dt).cuda().flatten(1)
    for x, one in ((kr, "k"), (vr, "v")):
        if cache == "fp4":
            codes, scales = to_fp4(x, getattr(c, one + "_scale"))
        for i, (_, b, pos) in enumerate(stored):
            page, slot = int(c.table[b, pos // 16]), pos % 16
            if cache == "fp4":
                want[one + "pool"][page, :, slot] = torch.from_numpy(codes[i]).cuda()
                want[one + "scale"][page, :, slot] = torch.from_numpy(scales[i]).cuda()
            else:
                want[one + "pool"][page, :, slot] = torch.from_numpy(x[i]).to(c.kpool.dtype).cuda().view(torch.uint8)
    q_out = torch.full_like(c.q, 777.0)
    ops.kv_append(c.kv, c.nr, c.k, c.v, rope=rope, q=c.q, q_out=q_out, heads=heads)
    ops.status()
    for n in names:
        got = raw(getattr(c, n))
        assert bool((got == want[n]).all()), (n, int((got != want[n]).sum()))
    assert bool((q_out == q_want).all())
    ko, vo = torch.full_like(c.k, 777.0), torch.full_like(c.v, 777.0)
    ops.kv_read(c.kv, c.nr, ko, vo)
    ops.status()
    for one, got in (("k", ko), ("v", vo)):
        w = torch.full_like(got, 777.0)
        for t, b, pos in stored:
            # a 4-bit value times the pool's scale is rounded to fp32 before it is rounded to the rows' type
            w[t] = c.cached(one, b, pos + 1)[:, pos].float().to(c.dt).flatten()
        assert bool((got == w).all())


@pytest.mark.parametrize("cache,rows", [("bf16", "f32"), ("fp4", "bf16"), ("f32", "f32")])
def test_append_strides_no_table_in_place(api, ops, cache, rows):
    """k, v and q as parts of one projection's rows, on odd boundaries; q rotated in place; without a table, rows as they are."""
    import torch
    heads, kv_heads, hd = 6, 2, 64
    for off in (0, 1):
        c = Case(api, [1, 9, 30], [7, 9, 50], heads, kv_heads, hd, cache, rows)
        wq, wk = heads * hd, kv_heads * hd
        buf = torch.zeros(c.rows * (wq + 2 * wk + 8) + off, dtype=c.dt, device="cuda")
        full = buf[off:].view(c.rows, wq + 2 * wk + 8)
        q, k, v = full[:, :wq], full[:, wq:wq + wk], full[:, wq + wk:wq + 2 * wk]
        for x, y in ((q, c.q), (k, c.k), (v, c.v)):
            x.copy_(y)
        rope = rope_table(50, hd)
        d = Case(api, [1, 9, 30], [7, 9, 50], heads, kv_heads, hd, cache, rows)
        q_out = torch.empty_like(d.q)
        ops.kv_append(d.kv, d.nr, d.k, d.v, rope=rope, q=d.q, q_out=q_out, heads=heads)
        ops.kv_append(c.kv, c.nr, k, v, rope=rope, q=q, q_out=q, heads=heads)
        assert bool((q == q_out).all())
        for n in ("kpool", "vpool"):
            assert bool((getattr(c, n).view(torch.uint8) == getattr(d, n).view(torch.uint8)).all())
        ko, vo = torch.empty_like(d.k), torch.empty_like(d.v)
        ops.kv_append(c.kv, c.nr, k, v)
        ops.kv_read(c.kv, c.nr, ko, vo)
        if cache != "fp4":
            assert bool((ko == k.to(c.kpool.dtype).to(c.dt)).all()) and bool((vo == v.to(c.kpool.dtype).to(c.dt)).all())
        ops.status()


def test_append_extremes(api, ops):
    """4 bits: values far above and below the pool's scale, infinities, zeros, and ties between codes."""
    import torch
    c = Case(api, [4], [4], 1, 1, 64, "fp4", "f32", k_scale=1.0, v_scale=1.0)
    c.k.zero_()
    c.k[0, :16] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6.0])
    c.k[1] = 1e30
    c.k[2] = 1e-30
    c.k[3] = math.inf
    c.v.copy_(-c.k)
    ops.kv_append(c.kv, c.nr, c.k, c.v)
    ko, vo = torch.empty_like(c.k), torch.empty_like(c.v)
    ops.kv_read(c.kv, c.nr, ko, vo)
    ties = [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, -6.0]
    assert ko[0, :16].tolist() == ties and (-vo[0, :16]).tolist() == ties
    assert bool((ko[1] == 6 * 448).all()) and bool((vo[1] == -6 * 448).all())
    assert bool((ko[2] == 0).all()) and bool((ko[3] == 6 * 448).all())
    assert bool((ko[0, 16:] == 0).all())


# ---- what the caller's data can have wrong -----------------------------------------------------------------------------
@pytest.mark.parametrize("cache,rows", [("bf16", "bf16"), ("fp4", "f32"), ("f32", "f32")])
def test_bad_data_is_reported(api, ops, cache, rows):
    import torch
    def fresh():
        return Case(api, [2, 3, 40], [20, 3, 60], 4, 2, 64, cache, rows)

    def refused(c, call, text):
        call(c)
        with pytest.raises(api.MlbError, match=text):
            ops.status()
        ops.status()

    def append(c):
        ops.kv_append(c.kv, c.nr, c.k, c.v)

    for bad in (-1, 10 ** 9):
        c = fresh()
        c.table[2, 2] = bad
        before = c.kpool.clone()
        refused(c, append, "page")
        touched = (c.kpool.view(torch.uint8) != before.view(torch.uint8)).flatten(1).any(1).nonzero().flatten().tolist()
        ok = set(c.table[0].tolist() + c.table[1].tolist() + c.table[2].tolist())
        assert set(touched) <= ok
        refused(c, lambda c: attend(ops, c), "page")
    c = fresh()
    want, tol = c.attention()
    c.kv_lens[1] = 10 ** 6
    out = torch.full((c.rows, c.heads * c.hd), 777.0, dtype=c.dt, device="cuda")
    refused(c, lambda c: attend(ops, c, out=out), "pt_stride")
    want[2:5] = math.nan
    check(out, want, tol)
    refused(c, append, "pt_stride")
    c = fresh()
    c.row_start[1] = 50
    refused(c, lambda c: attend(ops, c), "row_start")
    refused(c, append, "row_start")
    c = fresh()
    c.describe(max_rows=39)
    refused(c, lambda c: attend(ops, c), "max_rows")
    c = fresh()
    rope = rope_table(59, 64)
    refused(c, lambda c: ops.kv_append(c.kv, c.nr, c.k, c.v, rope=rope), "rotation")


def test_wrapper_refuses(api, ops):
    import torch
    c = Case(api, [1, 2], [5, 6], 4, 2, 64)
    out = torch.empty_like(c.q)
    with pytest.raises(ValueError):
        ops.attn_paged(c.kv, c.nr, c.q.half(), out, heads=4)
    with pytest.raises(ValueError):
        ops.attn_paged(c.kv, c.nr, c.q, out.float(), heads=4)
    with pytest.raises(ValueError):
        ops.attn_paged(c.kv, c.nr, c.q[:2], out, heads=4)
    with pytest.raises(ValueError):
        ops.attn_paged(c.kv, c.nr, c.q.cpu(), out, heads=4)
    with pytest.raises(api.MlbError):
        ops.attn_paged(c.kv, c.nr, c.q, out, heads=4, window=-3)
    with pytest.raises(ValueError):
        api.PagedKV(c.kpool, c.vpool[:, :1], c.table)
    with pytest.raises(api.MlbError):
        api.Ops(977)


# ---- together, as a server uses them -----------------------------------------------------------------------------------
@pytest.mark.parametrize("cache,rows", [("bf16", "bf16"), ("f32", "f32"), ("fp4", "bf16"), ("fp4", "f32"), ("bf16", "f32")])
def test_prompt_then_steps(api, ops, cache, rows):
    """Prompts in, then step after step: every step's attention is that of the formula over what kv_read says is cached, and the steps of a
    sequence equal one call for all of its rows."""
    import torch
    heads, kv_heads, hd, steps = 8, 2, 64, 20
    prompts = [37, 1, 90]
    total = [p + steps for p in prompts]
    c = Case(api, total, total, heads, kv_heads, hd, cache, rows)
    rope = rope_table(max(total), hd)
    q_rot = torch.empty_like(c.q)
    # all rows at once, on a second set of pools
    d = Case(api, total, total, heads, kv_heads, hd, cache, rows)
    ops.kv_append(d.kv, d.nr, d.k, d.v, rope=rope, q=d.q, q_out=q_rot, heads=heads)
    out = attend(ops, d, 30, 2, q=q_rot)
    check(out, *d.attention(30, 2, q=q_rot))
    first = np.concatenate([[0], np.cumsum(total)])
    for step in range(steps + 1):
        new = prompts if step == 0 else [1] * 3
        lens = [p + step for p in prompts]
        t = np.concatenate([np.arange(first[b] + lens[b] - new[b], first[b] + lens[b]) for b in range(3)]).tolist()
        nr = api.NewRows(torch.tensor(lens, dtype=torch.int32, device="cuda"), len(t), max_rows=max(new),
                         row_start=torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda") if step == 0 else None)
        q = torch.empty_like(c.q[t])
        o = torch.empty_like(q)
        ops.kv_append(c.kv, nr, c.k[t], c.v[t], rope=rope, q=c.q[t], q_out=q, heads=heads)
        ops.attn_paged(c.kv, nr, q, o, heads=heads, window=30, sinks=2)
        assert bool((q == q_rot[t]).all())
        want, tol = d.attention(30, 2, q=q_rot)
        assert float(((o.double() - want[t]).abs() - tol[t]).max()) <= 0
    ops.status()


@pytest.mark.parametrize("cache,rows", [("bf16", "bf16"), ("fp4", "f32")])
def test_captured_and_replayed(api, cache, rows):
    """A step captured into a graph and replayed while the lengths move on; a second handle on another stream at the same time."""
    import torch
    B, L0 = 5, 200
    own, other = api.Ops(0), api.Ops(0)
    c = Case(api, [1] * B, [L0 + 40] * B, 16, 4, 128, cache, rows, ragged=False)
    rope = rope_table(L0 + 40, 128)
    out, q = torch.empty_like(c.q), torch.empty_like(c.q)
    c.kv_lens.fill_(L0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def step(ops, stream):
        ops.kv_append(c.kv, c.nr, c.k, c.v, rope=rope, q=c.q, q_out=q, heads=16, stream=stream)
        ops.attn_paged(c.kv, c.nr, q, out, heads=16, window=100, sinks=4, stream=stream)

    with torch.cuda.stream(s):
        step(own, s.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(own, torch.cuda.current_stream().cuda_stream)
    e = Case(api, [1, 60], [900, 300], 8, 2, 64, cache, rows, seed=3)
    want_e, tol_e = e.attention(0, 0)
    s2 = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(10):
        c.kv_lens.fill_(L0 + 1 + i)
        torch.cuda.synchronize()
        g.replay()
        oe = torch.full_like(e.q, 777.0)
        s2.wait_stream(torch.cuda.current_stream())
        other.attn_paged(e.kv, e.nr, e.q, oe, heads=8, stream=s2.cuda_stream)
        torch.cuda.synchronize()
        c.lens = [L0 + 1 + i] * B
        check(out, *c.attention(100, 4, q=q))
        check(oe, want_e, tol_e)
    own.status()
    other.status(s2.cuda_stream)
    del g


@pytest.mark.parametrize("cache,rows", [("bf16", "bf16"), ("fp4", "bf16"), ("f32", "f32")])
def test_offsets_past_32_bits(api, ops, cache, rows):
    """Pages whose bytes, and elements, lie more than 2^32 from the pool's start."""
    import torch
    kv_heads, hd = 8, 128
    per = kv_heads * 16 * hd
    pages = ((1 << 32) + (1 << 28)) // per // (1 if cache != "fp4" else 1)
    if torch.cuda.mem_get_info()[0] < 2 * pages * per * 5:
        pytest.skip("not enough device memory")
    small = Case(api, [1, 150], [400, 170], 16, kv_heads, hd, cache, rows)
    want, tol = small.attention(100, 3)
    names = ["kpool", "vpool"] + (["kscale", "vscale"] if cache == "fp4" else [])
    for n in names:
        x = getattr(small, n)
        big = torch.empty((pages, *x.shape[1:]), dtype=x.dtype, device="cuda")
        big[pages - x.shape[0]:].view(torch.uint8).copy_(x.view(torch.uint8))
        setattr(small, n, big)
    small.table += pages - small.n_pages
    small.describe()
    check(attend(ops, small, 100, 3), want, tol)
    ops.kv_append(small.kv, small.nr, small.k, small.v)
    ko, vo = torch.empty_like(small.k), torch.empty_like(small.v)
    ops.kv_read(small.kv, small.nr, ko, vo)
    ops.status()
    if cache != "fp4":
        assert bool((ko == small.k).all()) and bool((vo == small.v).all())


def test_same_answer_as_the_decode_operator(api, ops):
    """On a cache that mlb_op_attn_decode reads too, without a window the two agree to fp32 rounding."""
    import torch
    lens = [1, 16, 250, 77]
    c = Case(api, [1] * 4, lens, 8, 2, 128, "bf16", "f32", ragged=False)
    out, ref = attend(ops, c), torch.empty_like(c.q)
    pos = c.kv_lens - 1
    rc = api.lib().mlb_op_attn_decode(c.kpool.data_ptr(), c.vpool.data_ptr(), api.DT_BF16, c.table.data_ptr(), c.table.shape[1], c.n_pages,
                                      pos.data_ptr(), c.q.data_ptr(), None, ref.data_ptr(), 4, 8, 2, 128, 3, None)
    assert rc == 0
    assert float((out - ref).abs().max()) < 2e-5


# ---- sizes at which the work is dealt out in another way ---------------------------------------------------------------
@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("batch,kv_heads", [(40, 2), (300, 1), (700, 2)])
def test_short_sequences_beside_long_ones(api, ops, cache, rows, batch, kv_heads):
    """Batches on both sides of a CTA's 256 threads, few and many items for each CTA; shares with several short items, long items in many shares."""
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 60, size=batch)
    lens[rng.integers(0, batch, size=3)] = rng.integers(2000, 6000, size=3)
    c = Case(api, [1] * batch, lens.tolist(), 4 * kv_heads, kv_heads, 64, cache, rows, ragged=False)
    for window, sinks in ((0, 0), (700, 20)):
        check(attend(ops, c, window, sinks), *c.attention(window, sinks))
    ops.status()


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(3, 1, 64), (16, 4, 128), (12, 12, 64)])
def test_append_of_many_rows(api, ops, cache, rows, heads, kv_heads, hd):
    """Several rows for a CTA: the same bits as sequence by sequence, a row for a CTA each."""
    import torch
    new, lens = [900, 0, 1, 1100, 3, 57, 1000, 640, 1013], [900, 7, 1, 1500, 2, 57, 1300, 640, 1020]
    for steps in (1, 4):
        n, L = (new, lens) if steps == 1 else ([x * 4 for x in new], [x * 4 for x in lens])
        c, d = (Case(api, n, L, heads, kv_heads, hd, cache, rows, extra_rows=5) for _ in range(2))
        rope = rope_table(max(L), hd)
        q_out, q_ref = torch.full_like(c.q, 777.0), torch.full_like(c.q, 777.0)
        outs, refs = ([torch.full_like(c.k, 777.0) for _ in range(2)] for _ in range(2))
        ops.kv_append(c.kv, c.nr, c.k, c.v, rope=rope, q=c.q, q_out=q_out, heads=heads)
        ops.kv_read(c.kv, c.nr, *outs)
        t = 0
        for b, (m, length) in enumerate(zip(n, L)):
            for i in range(0, m, 500):
                k = min(500, m - i)
                kv = api.PagedKV(d.kpool, d.vpool, d.table[b:b + 1].contiguous(), kscale=d.kscale, vscale=d.vscale, k_scale=d.k_scale, v_scale=d.v_scale)
                nr = api.NewRows(torch.tensor([length - m + i + k], dtype=torch.int32, device="cuda"), k,
                                 row_start=torch.tensor([0, k], dtype=torch.int32, device="cuda"))
                s = slice(t + i, t + i + k)
                ops.kv_append(kv, nr, d.k[s], d.v[s], rope=rope, q=d.q[s], q_out=q_ref[s], heads=heads)
                ops.kv_read(kv, nr, refs[0][s], refs[1][s])
            t += m
        ops.status()
        assert bool((q_out == q_ref).all())
        for one in ["kpool", "vpool"] + (["kscale", "vscale"] if cache == "fp4" else []):
            assert bool((getattr(c, one).view(torch.uint8) == getattr(d, one).view(torch.uint8)).all()), one
        for x, y in zip(outs, refs):
            assert bool((x == y).all())


@pytest.mark.parametrize("cache,rows", TYPES)
def test_calls_in_a_row(api, ops, cache, rows):
    """Calls of one handle behind one another, none waited for: each has the scratch to itself."""
    cases = [Case(api, [1, 200, 1, 40], [4000, 300, 77, 2000], 8, 2, 64, cache, rows, seed=1), Case(api, [1] * 70, [500] * 70, 8, 2, 128, cache, rows, ragged=False, seed=2),
             Case(api, [3, 1], [9000, 6000], 8, 2, 128, cache, rows, seed=3)]
    alone = [attend(ops, c, 900, 4) for c in cases]
    ops.status()
    for c, out in zip(cases, alone):
        check(out, *c.attention(900, 4))
    for _ in range(5):
        again = [attend(ops, c, 900, 4) for c in cases]
        for a, b in zip(alone, again):
            assert bool((a == b).all())
    ops.status()


@pytest.mark.parametrize("cache", ["bf16", "fp4", "f32"])
def test_captured_prompts(api, ops, cache):
    """Prompts beside single tokens, captured once and replayed with other lengths and row counts within the same rows."""
    import torch
    c = Case(api, [1, 300, 4, 90], [700, 900, 350, 95], 8, 2, 64, cache, "bf16", extra_rows=3)
    c.describe()
    out = torch.empty_like(c.q)
    s = torch.cuda.Stream()
    ops.attn_paged(c.kv, c.nr, c.q, out, heads=8, window=333, sinks=9)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out.fill_(777.0)
        ops.attn_paged(c.kv, c.nr, c.q, out, heads=8, window=333, sinks=9, stream=torch.cuda.current_stream().cuda_stream)
    for new, lens in (([1, 300, 4, 90], [700, 900, 350, 95]), ([100, 1, 200, 0], [600, 20, 201, 3]), ([1, 1, 1, 1], [1, 2, 3, 17]), ([0, 0, 0, 398], [5, 5, 5, 96 - 1])):
        if lens[3] < new[3]:
            lens[3] = 95                          # rows before position 0 are zeros
        c.new, c.lens = new, lens
        c.row_start.copy_(torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32))
        c.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        for _ in range(2):
            g.replay()
        torch.cuda.synchronize()
        check(out, *c.attention(333, 9))
    ops.status()
    del g


def test_out_is_not_q(api, ops):
    import torch
    c = Case(api, [1, 2], [5, 6], 4, 2, 64)
    with pytest.raises(api.MlbError, match="may not be q"):
        ops.attn_paged(c.kv, c.nr, c.q, c.q, heads=4)
    with pytest.raises(ValueError, match="q_out"):
        ops.kv_append(c.kv, c.nr, c.k, c.v, q=c.q, heads=4)
    with pytest.raises(api.MlbError, match="stride"):
        ops.kv_append(c.kv, c.nr, c.k[:1].expand(3, -1), c.v)
    assert torch.cuda.current_device() == 0
