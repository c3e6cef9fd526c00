"""GPU: paged operators at the ends of their ranges: weights over a wide range, pools of many rows, values that are no numbers."""
import math

import numpy as np
import pytest

from test_gpu_paged import TYPES, U, U16, Case, attend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(built_lib):
    from mini_llm_cuda_b200 import api as _api
    return _api


@pytest.fixture(scope="module")
def ops(api):
    return api.Ops(0)


# ---- weights over a wide range -----------------------------------------------------------------------------------------
def first_key_takes_all(c, above):
    """Scores of about `above` powers of two at position 0 of every sequence, whose value is 0.001, and of -1, 0 or 1 elsewhere: the output is made of
    the small weights. A score has two products, the rest are zeros."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    first = c.table[:, 0].long()
    sign = torch.randint(0, 3, c.kpool.shape[:3], generator=g, device="cuda")
    c.kpool.zero_()
    if c.cache == "fp4":
        c.kscale.copy_(torch.ones(c.kscale.shape, device="cuda"))
        c.kpool[..., 0] = torch.tensor([0x00, 0x20, 0xa0], dtype=torch.uint8, device="cuda")[sign]      # dim 1: 0, 1, -1
        c.kpool[first, :, 0, 0] = 0x02                                                                  # dim 0: 1
        c.vpool[first, :, 0] = 0x11
        c.vscale[first, :, 0] = torch.full((), 2.0 ** -9, device="cuda").to(torch.float8_e4m3fn)
    else:
        c.kpool[..., 1] = (sign - 1).to(c.kpool.dtype)
        c.kpool[first, :, 0, 1] = 0
        c.kpool[first, :, 0, 0] = 1
        c.vpool[first, :, 0] = 0.001
    q = torch.zeros(c.rows, c.heads, c.hd, device="cuda")
    q[..., 0] = above * math.log(2) * math.sqrt(c.hd) * (1 + 0.01 * torch.arange(c.heads, device="cuda"))
    q[..., 1] = 0.7 * math.sqrt(c.hd)
    c.q = q.flatten(1).to(c.dt)


def small_weights(c, out):
    """Largest error of the output over its bound, relative to the sum of w |v| and not to the largest value."""
    import torch
    H, D, KH, worst, r0 = c.heads, c.hd, c.kv_heads, 0.0, 0
    for b, (n, L) in enumerate(zip(c.new, c.lens)):
        q = c.q[r0:r0 + n].double().reshape(n, KH, H // KH, D).permute(1, 2, 0, 3)
        K, V = c.cached("k", b, L), c.cached("v", b, L)
        hidden = torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None]
        s = (q @ K[:, None].transpose(-1, -2) / math.sqrt(D)).masked_fill(hidden, -math.inf)
        w = torch.softmax(s, dim=-1)
        o, size = w @ V[:, None], w @ V[:, None].abs()
        # An exponent of 2 (a score times log2 e) has up to four roundings of two products and three factors, relative to a magnitude of `most`, and
        # so has the reference that is taken off it; the exponential two steps. A sum is taken by 16 positions, whose products may be cut off where they are added, a
        # whole step twice, and 20 steps where partial sums are put together and divided; the pieces of a number leave out half a step each.
        most = float((q.abs() @ K[:, None].abs().transpose(-1, -2) / math.sqrt(D)).amax())
        t = size * U * (2 * 4 * most + 4 + 4 * (L / 16 + 1) + 20 + 6)
        if c.dt == torch.bfloat16:
            t = t + 1.1 * U16 * (o.abs() + size)             # as the documentation has it: probabilities may be rounded to bf16, the result is
        got = out[r0:r0 + n].double().reshape(n, KH, H // KH, D).permute(1, 2, 0, 3)
        worst = max(worst, float(((got - o).abs() / t).max()))
        r0 += n
    return worst


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,batch,length", [(1, 1, 1700), (1, 600, 200), (3, 2, 1700), (40, 2, 1700), (1, 3, 15)])
def test_small_weights_count(api, ops, cache, rows, hd, new, batch, length):
    """One key far above the rest: what the rest add up to is as exact as if they stood alone (a first position that takes most of the weight and
    brings next to nothing is what trained models have)."""
    c = Case(api, [new] * batch, [length] * batch, 4, 2, hd, cache, rows, k_scale=1.0, v_scale=1.0)
    for above in (0, 13, 20, 27, 40):
        first_key_takes_all(c, above)
        c.describe()
        worst = small_weights(c, attend(ops, c))
        assert worst <= 1, f"{worst:.3g} of the bound, a key 2^{above} above the rest"
    ops.status()


# ---- pools of more than 2^31 rows --------------------------------------------------------------------------------------
def test_4_bit_pools_may_have_more_rows(api, ops):
    """2^31 rows of a head fit the device at 4 bits. The pool described here is that large, the one behind it holds the pages that the table names."""
    import torch
    c = Case(api, [1, 90], [300, 120], 2, 1, 64, "fp4", "bf16")
    c.kv.struct.num_pages = (1 << 27) + 1
    want, tol = c.attention(50, 3)
    out = attend(ops, c, 50, 3)
    ops.status()
    assert float(((out.double() - want).abs() - tol).max()) <= 0
    # of bf16 it is refused where prompts may come, before anything is written
    c = Case(api, [1, 90], [300, 120], 2, 1, 64, "bf16", "bf16")
    c.kv.struct.num_pages = (1 << 27) + 1
    out = torch.full_like(c.q, 777.0)
    with pytest.raises(api.MlbError, match="2\\^31"):
        attend(ops, c, 50, 3, out=out)
    assert bool((out == 777.0).all())


# ---- values that are no numbers ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("heads,hd", [(2, 64), (8, 128)])
@pytest.mark.parametrize("new,length", [(1, 300), (3, 77), (50, 90)])
def test_one_value_is_no_number(api, ops, cache, rows, heads, hd, new, length):
    """An infinite value in one dim of one position (4 bits: a NaN scale, sixteen dims): the other dims, and rows that do not see the position, are as
    if it were not there, and those that see it get no number in that dim."""
    import torch
    c = Case(api, [new], [length], heads, 2, hd, cache, rows)
    for at in (length - new + new // 2, 20):
        page, slot = int(c.table[0, at // 16]), at % 16
        if cache == "fp4":
            before = c.vscale.view(torch.uint8)[page, 1, slot, 2].clone()
            c.vscale.view(torch.uint8)[page, 1, slot, 2] = 0x7f
            dims = range(32, 48)
        else:
            before = c.vpool[page, 1, slot, 33].clone()
            c.vpool[page, 1, slot, 33] = math.inf
            dims = range(33, 34)
        want, tol = c.attention()
        out = attend(ops, c).double().reshape(new, 2, heads // 2, hd)
        sees = torch.arange(length - new, length, device="cuda") >= at
        hit = torch.zeros(new, 2, heads // 2, hd, dtype=torch.bool, device="cuda")
        hit[:, 1, :, dims.start:dims.stop] = sees[:, None, None]
        assert not bool(torch.isfinite(out[hit]).any())
        if cache != "fp4":
            assert bool((out[hit] == math.inf).all())
        over = (out - want.reshape(out.shape)).abs() - tol.reshape(out.shape)
        assert float(over[~hit].max()) <= 0
        if cache == "fp4":
            c.vscale.view(torch.uint8)[page, 1, slot, 2] = before
        else:
            c.vpool[page, 1, slot, 33] = before
    ops.status()


@pytest.mark.parametrize("cache,rows", [("bf16", "bf16"), ("f32", "f32"), ("fp4", "bf16"), ("fp4", "f32")])
@pytest.mark.parametrize("new,length", [(1, 20000), (1000, 1000)])
def test_a_row_without_an_answer_ends_early(api, ops, cache, rows, new, length):
    """A NaN among the first keys: nothing that follows can make the rows numbers, so they do not cost what a row done by hand does (over 300 times the
    call for these sizes, and 1 to 5 times where it ends with the answer)."""
    import torch

    def best():
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            out = attend(ops, c)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times), out

    c = Case(api, [new], [length], 16, 4, 128, cache, rows)
    clean, _ = best()
    page = int(c.table[0, 0])
    if cache == "fp4":
        c.kscale.view(torch.uint8)[page, :, 3, 0] = 0x7f
    else:
        c.kpool[page, :, 3, 7] = math.nan
    bad, out = best()
    assert bool(torch.isnan(out[max(0, 3 - (length - new)):]).all()) and bool(torch.isfinite(out[:max(0, 3 - (length - new))]).all())
    assert bad < 40 * clean, (bad, clean)


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 3, 90])
def test_hidden_scales_hold_no_numbers(api, ops, rows, new):
    """4 bits: NaN scales at positions that no row sees, as unused slots of a fresh page may have them."""
    import torch
    lens = [new + 200, new + 37, new, new + 129]
    window, sinks = 20, 5
    c = Case(api, [new] * 4, lens, 8, 2, 128, "fp4", rows)
    want, tol = c.attention(window, sinks)
    hidden = torch.ones(c.n_pages, 16, dtype=torch.bool, device="cuda")
    for b, L in enumerate(lens):
        for j in range(L):
            if j < sinks or j > L - new - window:
                hidden[int(c.table[b, j // 16]), j % 16] = False
    bad = torch.tensor([0x7f, 0xff], dtype=torch.uint8, device="cuda")
    for n, scale in enumerate((c.kscale, c.vscale)):
        v = scale.view(torch.uint8).permute(0, 2, 1, 3)
        v[hidden] = bad[(torch.arange(int(hidden.sum()), device="cuda") + n) % 2][:, None, None].expand(-1, c.kv_heads, 8)
    out = attend(ops, c, window, sinks).double()
    assert bool(torch.isfinite(out).all())
    assert float(((out - want).abs() - tol).max()) <= 0
    ops.status()


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("heads,hd", [(2, 64), (8, 128)])
@pytest.mark.parametrize("new,length", [(3, 60), (40, 60), (200, 260)])
def test_a_later_row_sees_no_scale(api, ops, rows, heads, hd, new, length):
    """4 bits: a position with NaN scales that later rows see and earlier ones do not."""
    import torch
    c = Case(api, [new], [length], heads, 2, hd, "fp4", rows)
    want, tol = c.attention()
    at = length - new // 2 - 1
    page, slot, before = int(c.table[0, at // 16]), at % 16, at - (length - new)
    for scale in (c.vscale, c.kscale):
        scale.view(torch.uint8)[page, :, slot] = 0xff
        out = attend(ops, c).double()
        assert float(((out - want).abs() - tol)[:before].max()) <= 0
        assert bool(torch.isnan(out[before:]).all())


def test_4_bit_offsets_past_32_bits(api, ops):
    """Codes more than 2^32 bytes from the pool's start: appended, read and attended to as in a small pool."""
    import torch
    kv_heads, hd = 8, 128
    pages = ((1 << 32) + (1 << 27)) // (kv_heads * 16 * hd // 2)
    if torch.cuda.mem_get_info()[0] < 3 * pages * kv_heads * 16 * hd:
        pytest.skip("not enough device memory")
    small, large = (Case(api, [1, 150], [400, 170], 16, kv_heads, hd, "fp4", "bf16", seed=9) for _ in range(2))
    n = small.n_pages
    names = ["kpool", "vpool", "kscale", "vscale"]
    for name in names:
        x = getattr(large, name)
        big = torch.zeros((pages, *x.shape[1:]), dtype=torch.uint8, device="cuda")
        big[pages - n:].copy_(x.view(torch.uint8))
        setattr(large, name, big if name.endswith("pool") else big.view(x.dtype))
    large.table += pages - n
    large.describe()
    read = []
    for c in (small, large):
        out = attend(ops, c, 100, 3)
        ops.kv_append(c.kv, c.nr, c.k, c.v)
        ko, vo = torch.empty_like(c.k), torch.empty_like(c.v)
        ops.kv_read(c.kv, c.nr, ko, vo)
        read.append((out, ko, vo))
    ops.status()
    for x, y in zip(*read):
        assert bool((x == y).all())
    for name in names:
        x, y = (getattr(c, name).view(torch.uint8) for c in (small, large))
        assert bool((x == y[pages - n:]).all()) and not bool(y[:pages - n].any())


# ---- every position once -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("kind", ["one", "few", "many", "crowd", "rows", "prompts"])
def test_every_position_counts_once(api, ops, cache, rows, heads, kv_heads, hd, kind):
    """Queries of zeros weigh all that is visible alike. Values count: one dim holds ones at every hd-th position (or page), the next dim at the ones after
    them, so that a position or page left out or taken twice, at any share's, tile's or page's border, is off by a whole number."""
    import torch
    rng = np.random.default_rng(11)
    new, lens, ragged = {
        "one": ([1], [5003], False),
        "few": ([1] * 9, [3333, 1, 16, 2049, 700, 17, 4096, 31, 1200], False),
        "many": ([1] * 70, rng.integers(1, 1500, size=70).tolist(), False),
        "crowd": ([1] * 640, rng.integers(1, 300, size=640).tolist(), False),
        "rows": ([1, 3, 0, 4, 2, 8, 1], [2222, 1003, 5, 64, 18, 3000, 1], True),
        "prompts": ([130, 1, 33, 257, 64], [900, 40, 1033, 257, 2000], True),
    }[kind]
    c = Case(api, new, lens, heads, kv_heads, hd, cache, rows, ragged=ragged, k_scale=1.0, v_scale=1.0)
    c.q.zero_()
    if cache == "fp4":
        c.vscale.copy_(torch.ones(c.vscale.shape, device="cuda"))
    t = torch.arange(max(lens), device="cuda")
    for which in (t % hd, t // 16 % hd):
        c.vpool.zero_()
        ones = (which[:, None] == torch.arange(hd, device="cuda")).double()
        for b, L in enumerate(lens):
            v = ones[:L]
            if cache == "fp4":
                v = (v[:, 0::2] * 2 + v[:, 1::2] * 32).to(torch.uint8)               # code 2 is 1
            full = torch.zeros((L + 15) // 16 * 16, v.shape[1], dtype=c.vpool.dtype, device="cuda")
            full[:L] = v.to(c.vpool.dtype)
            c.vpool[c.table[b, :(L + 15) // 16].long()] = full.reshape(-1, 1, 16, v.shape[1])
        for window, sinks in ((0, 0), (1000, 37), (77, 3)):
            out = attend(ops, c, window, sinks).double().reshape(c.rows, heads, hd)
            r0 = 0
            for n, L in zip(new, lens):
                p = torch.arange(L - n, L, device="cuda")[:, None]
                sees = t[None, :L] <= p
                if window:
                    sees &= (t[None, :L] > p - window) | (t[None, :L] < sinks)
                count, total = sees.double() @ ones[:L], sees.sum(1).double()
                off = (out[r0:r0 + n] * total[:, None, None] - count[:, None]).abs()
                # equal weights are whole powers of two and sums of ones exact: the answer is rounded once or twice, and so off by less than a half
                assert n == 0 or float(off.max()) < 0.5, (kind, n, L, window, float(off.max()))
                r0 += n
    ops.status()


@pytest.mark.parametrize("cache", ["f32", "bf16", "fp4"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,batch,length", [(1, 1, 2900), (1, 600, 130), (4, 3, 700), (70, 2, 700)])
def test_fp32_rows_to_fp32(api, ops, cache, hd, new, batch, length):
    """fp32 rows, relative to the sum of w |v| of each number: an operand rounded to bf16 on the way would show (some 2^-9 of a score of 3, which the sum over
    some hundred positions leaves a tenth of)."""
    import torch
    c = Case(api, [new] * batch, [length] * batch, 4, 2, hd, cache, "f32")
    if cache == "fp4":                               # values of about the size of the others'
        c.k_scale, c.v_scale = 0.02, 0.02
        c.describe()
    out = attend(ops, c, length // 2, 3)
    KH, G, r0 = c.kv_heads, c.heads // c.kv_heads, 0
    for b, (n, L) in enumerate(zip(c.new, c.lens)):
        q = c.q[r0:r0 + n].double().reshape(n, KH, G, hd).permute(1, 2, 0, 3)
        K, V = c.cached("k", b, L), c.cached("v", b, L)
        p, j = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")[None]
        s = (q @ K[:, None].transpose(-1, -2) / math.sqrt(hd)).masked_fill((j > p) | (j <= p - length // 2) & (j >= 3), -math.inf)
        w = torch.softmax(s, dim=-1)
        o, size = w @ V[:, None], w @ V[:, None].abs()
        most = (q.abs() @ K[:, None].abs().transpose(-1, -2) / math.sqrt(hd)).amax(-1, keepdim=True)
        # A score is taken in hd / 16 steps of up to six products of pieces, each of which may cut off where it adds (a whole step, 2 U, of at most `most`), has
        # three factors, and 4-bit queries' 22 bits (4 U); so has the maximum that is taken off it. The sum over weights: L / 16 such steps. The exponential,
        # the division and the joining of partial sums: 30.
        t = size * U * (2 * (2 * 6 * (hd / 16) + 4 + 4) * most + 2 * 6 * (L / 16 + 1) + 30)
        got = out[r0:r0 + n].double().reshape(n, KH, G, hd).permute(1, 2, 0, 3)
        assert float(((got - o).abs() / t).max()) <= 1
        r0 += n
    ops.status()


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [1, 4, 7])
def test_weights_next_to_a_band(api, ops, rows, heads):
    """4 bits, one key far above the rest and all others alike, at every hundredth of a power of two around the border of the bands that halves are taken
    in (2^-26 of the largest): what the others add up to is there at each."""
    import torch
    L, above = 500, torch.arange(24.0, 30.0, 0.01, device="cuda")
    c = Case(api, [1] * len(above), [L] * len(above), heads, 1, 64, "fp4", rows, k_scale=1.0, v_scale=1.0, ragged=False)
    c.table[:] = c.table[0]
    first = int(c.table[0, 0])
    c.kpool.zero_()
    c.kscale.copy_(torch.ones(c.kscale.shape, device="cuda"))
    c.kpool[first, :, 0, 0] = 0x02
    c.vpool[first, :, 0] = 0
    c.q.zero_()
    c.q.view(len(above), heads, 64)[:, :, 0] = (above * math.log(2) * 8)[:, None].to(c.dt)
    out = attend(ops, c).double().reshape(len(above), heads, 64)
    x = c.q.view(len(above), heads, 64)[:, :, 0].double() / 8
    v = c.cached("v", 0, L)[0].sum(0)                # of 499 equal weights
    want = torch.exp(-x)[..., None] * v / (1 + (L - 1) * torch.exp(-x))[..., None]
    size = torch.exp(-x)[..., None] * c.cached("v", 0, L)[0].abs().sum(0)
    # as small_weights: two factors of one product, the reference's, the exponential; sums of L / 16 steps; bf16 rows: 11 bits of a weight and the result's 8
    t = size * U * (2 * 4 * 21 + 4 + 4 * (L / 16 + 1) + 20 + 6)
    if rows == "bf16":
        t = t + 1.1 * U16 * (want.abs() + size)
    assert float(((out - want).abs() / t).max()) <= 1
    ops.status()


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("new", [1, 3, 70])
def test_padding_rows_are_zeros_whatever_their_gates(api, ops, cache, rows, new):
    """A row before position 0 attends to nothing and is 0, though its gate and query were never written."""
    import torch
    lens = [max(0, new - 2), new + 20, 0]
    c = Case(api, [new] * 3, lens, 4, 2, 64, cache, rows)
    gate = torch.rand(c.rows, 4 * 64, device="cuda")
    want, tol = c.attention(30, 2, gate=gate)
    row = torch.arange(new, device="cuda")
    padding = torch.cat([row < new - n for n in lens])
    gate[padding] = torch.tensor([math.nan, math.inf, -math.inf, math.nan], device="cuda").repeat(64)
    c.q[padding] = math.nan
    out = attend(ops, c, 30, 2, gate=gate).double()
    assert bool((out[padding] == 0).all())
    assert float(((out - want).abs() - tol)[~padding].max()) <= 0
    ops.status()


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("new", [1, 5, 90])
def test_negative_scale(api, ops, cache, rows, new):
    c = Case(api, [new, new], [new + 200, new], 8, 2, 64, cache, rows)
    for scale in (-0.2, 1e-3):
        want, tol = c.attention(100, 3, scale=scale)
        # (the bound counts the scores' size by their sign)
        size = c.attention(100, 3, scale=abs(scale))[1]
        out = attend(ops, c, 100, 3, scale=scale).double()
        assert float(((out - want).abs() - tol.abs().maximum(size)).max()) <= 0
    ops.status()


@pytest.mark.parametrize("cache,rows", TYPES)
def test_4096_sequences(api, ops, cache, rows):
    """The most a call takes, many of them empty."""
    rng = np.random.default_rng(3)
    lens = (rng.integers(0, 40, size=4096) * (rng.random(4096) < 0.6)).tolist()
    c = Case(api, [1] * 4096, lens, 2, 1, 64, cache, rows, ragged=False)
    out = attend(ops, c, 20, 2).double()
    ops.status()
    pick = rng.choice(4096, size=300, replace=False).tolist() + [0, 4095]
    for b in pick:
        d = Case.__new__(Case)
        d.__dict__.update(c.__dict__)
        d.new, d.lens, d.rows, d.table, d.q = [1], [lens[b]], 1, c.table[b:b + 1], c.q[b:b + 1]
        want, tol = d.attention(20, 2)
        assert float(((out[b:b + 1] - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("cache", ["f32", "bf16", "fp4"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,batch,length", [(1, 1, 6000), (1, 300, 900), (40, 2, 1500)])
def test_fp32_error_as_a_whole(api, ops, cache, hd, new, batch, length):
    """fp32 rows: the error of all numbers together, against that of the same formula in plain fp32 torch operations. Both round at random, within half a step of what
    they add to; cutting off instead, a whole step always to the same side, gives several times as much. Twice the plain form's is allowed."""
    import torch
    c = Case(api, [new] * batch, [length] * batch, 4, 2, hd, cache, "f32", seed=4)
    if cache == "fp4":
        c.k_scale, c.v_scale = 0.02, 0.02
        c.describe()
    out = attend(ops, c)
    KH, G, r0, mine, plain = c.kv_heads, c.heads // c.kv_heads, 0, 0.0, 0.0
    for b, (n, L) in enumerate(zip(c.new, c.lens)):
        q = c.q[r0:r0 + n].double().reshape(n, KH, G, hd).permute(1, 2, 0, 3)
        K, V = c.cached("k", b, L)[:, None], c.cached("v", b, L)[:, None]
        hidden = torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None]
        forms = []
        for t in (torch.float64, torch.float32):
            s = (q.to(t) @ K.to(t).transpose(-1, -2) * (1 / math.sqrt(hd))).masked_fill(hidden, -math.inf)
            forms.append((torch.softmax(s, dim=-1) @ V.to(t)).double())
        got = out[r0:r0 + n].double().reshape(n, KH, G, hd).permute(1, 2, 0, 3)
        mine += float(((got - forms[0]) ** 2).sum())
        plain += float(((forms[1] - forms[0]) ** 2).sum())
        r0 += n
    assert mine <= 4 * plain, (math.sqrt(mine / plain))
    ops.status()


@pytest.mark.parametrize("cache,rows", TYPES)
@pytest.mark.parametrize("new", [1, 6, 60])
def test_scores_past_fp32_steps_of_one(api, ops, cache, rows, new):
    """Scores of some 10^8, where fp32's own steps are 8 and more: the largest takes all the weight; with its sign turned it has none."""
    import torch
    L = 300 + new
    c = Case(api, [new], [L], 4, 2, 64, cache, rows)
    key = 3                                             # slot 7 of this page stands out, by dim 0
    c.kpool.zero_()
    if cache == "fp4":
        c.kscale.copy_(torch.ones(c.kscale.shape, device="cuda"))
        c.kpool[c.table[0, key].long(), :, 7, 0] = 0x02
        c.k_scale = 1.0
    else:
        c.kpool[c.table[0, key].long(), :, 7, 0] = 1
    c.describe()
    c.q.zero_()
    c.q.view(new, 4, 64)[:, :, 0] = 1e9
    want = c.cached("v", 0, L)[:, key * 16 + 7].repeat_interleave(2, 0)[None].expand(new, -1, -1)
    out = attend(ops, c).double().view(new, 4, 64)
    t = want.abs() * (U16 * 1.1 * 2 if rows == "bf16" else U * 40)
    assert float(((out - want).abs() - t).max()) <= 0
    c.q.neg_()                                          # now that one is out, and all others weigh the same
    out = attend(ops, c).double().view(new, 4, 64)
    for i in range(new):
        keep = torch.arange(L - new + i + 1, device="cuda") != key * 16 + 7
        v = c.cached("v", 0, L - new + i + 1)[:, keep]
        mean, size = (x.mean(1).repeat_interleave(2, 0) for x in (v, v.abs()))
        t = size * U * (4 * (L / 16 + 1) + 40) + (1.1 * U16 * (size + mean.abs()) if rows == "bf16" else 0)
        assert float(((out[i] - mean).abs() - t).max()) <= 0
    ops.status()
