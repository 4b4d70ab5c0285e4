"""GPU parity of the paged 8-bit key/value cache (uwc_amd.kv) against its definitions in 64 bits: appending,
attention, reading back, at odd sizes, ragged and empty sequences, masks that leave rows empty, strides, and
numbers at the types' borders."""
import math

import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def check(got, want, tol, what=""):
    if not want.numel():
        return
    err = (got.double() - want).abs()
    worst = (err - tol).max().item()
    assert not torch.isnan(err).any() and worst <= 0, f"{what}: off by {worst:.3g} more than its bound"


def problem(dev, new, lens, H, Hkv, hd, page, dtype, seed=0, q_scale=1.5, pad=0, width=None):
    g = torch.Generator().manual_seed(seed)
    table, pages = R.make_table(lens, page, g, dev, width=width)
    cache = R.make_cache(pages, Hkv, hd, page, g, dev)
    q = (q_scale * torch.randn((sum(new) + pad, H, hd), generator=g)).to(dtype).to(dev)
    return cache, q, table, R.ints(lens, dev), R.cumulative(new, dev)


SHAPES = [  # new, lens, H, Hkv, hd, page, dtype
    ([1], [1], 1, 1, 128, 16, BF),
    ([1], [778], 16, 8, 128, 64, BF),
    ([1, 1, 1], [17, 64, 333], 8, 8, 64, 32, HF),
    ([1, 1], [65, 2500], 32, 8, 128, 128, HF),
    ([5, 5], [5, 900], 56, 8, 128, 16, BF),
    ([2, 0, 7, 1], [130, 40, 7, 64], 12, 4, 64, 16, BF),
    ([64], [64], 2, 1, 32, 32, HF),
    ([63, 129, 1], [63, 200, 1], 6, 2, 128, 64, BF),
    ([200, 31], [211, 500], 14, 2, 64, 128, HF),
    ([300], [1111], 7, 1, 128, 32, BF),
    ([257, 300], [257, 1400], 8, 8, 128, 16, HF),
    ([90, 700], [90, 700], 16, 2, 64, 64, BF),
    ([33], [700], 21, 7, 32, 16, BF),
]


@pytest.mark.parametrize("new,lens,H,Hkv,hd,page,dtype", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (33, 4), (100, 20), (64, 70)])
def test_attend_matches_definition(dev, new, lens, H, Hkv, hd, page, dtype, window, sinks):
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, new, lens, H, Hkv, hd, page, dtype, seed=len(new) + H)
    want, tol = R.attend(cache, q, table, L, cu, window, sinks)
    got = kv.attend(cache, q, table, L, cu=cu, max_new=max(new), max_len=max(lens), window=window, sinks=sinks)
    assert got.shape == q.shape and got.dtype == dtype
    check(got, want, tol)
    # bounds that say nothing, or the wrong thing, change the split alone
    check(kv.attend(cache, q, table, L, cu=cu, window=window, sinks=sinks), want, tol, "no bounds")
    check(kv.attend(cache, q, table, L, cu=cu, max_new=1, max_len=1, window=window, sinks=sinks), want, tol, "low bounds")
    if all(n == 1 for n in new):
        check(kv.attend(cache, q, table, L, max_len=max(lens), window=window, sinks=sinks), want, tol, "without cu")


@pytest.mark.parametrize("B,longest,H,Hkv,hd,window,sinks,dtype", [(1, 40000, 32, 8, 128, 0, 0, HF), (3, 9000, 8, 1, 64, 4096, 4, BF),
                                                                  (40, 3000, 4, 4, 128, 0, 0, BF), (1, 70001, 3, 1, 32, 8192, 20, BF)])
def test_attend_long_decode(dev, B, longest, H, Hkv, hd, window, sinks, dtype):
    """Keys split over workgroups and joined; the same bits each time."""
    from uwc_amd import kv
    lens = [longest - 61 * b for b in range(B)]
    cache, q, table, L, cu = problem(dev, [1] * B, lens, H, Hkv, hd, 16 if window else 64, dtype, seed=B)
    want, tol = R.attend(cache, q, table, L, cu, window, sinks)
    got = kv.attend(cache, q, table, L, max_len=longest, window=window, sinks=sinks)
    check(got, want, tol)
    assert torch.equal(got, kv.attend(cache, q, table, L, max_len=longest, window=window, sinks=sinks))


@pytest.mark.parametrize("new", [1, 70])
def test_attend_rows_of_no_sequence_and_rows_that_see_nothing(dev, new):
    """Padding rows, and queries before the sequence's first token (lens below new), are zeros."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, [new, new], [200, 300], 4, 2, 64, 16, BF, pad=133)
    L[1] = new // 2
    got = kv.attend(cache, q, table, L, cu=cu, max_new=new, max_len=300)
    check(got[:2 * new], *(x[:2 * new] for x in R.attend(cache, q, table, L, cu)))
    assert not got[2 * new:].any()
    assert not got[new:2 * new - new // 2].any()


@pytest.mark.parametrize("new", [1, 80])
def test_attend_pages_that_are_not_needed(dev, new):
    """Freed pages (entries that name no page, pages whose scales are NaN or infinite) outside every row's window."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, [new], [1000], 8, 4, 128, 16, HF, width=70)
    window, sinks = 100, 5
    want, tol = R.attend(cache, q, table, L, cu, window, sinks)
    for col in range(1, (1000 - new - window + 1) // 16):
        page = int(table[0, col])
        cache[2][page], cache[3][page] = math.nan, math.inf
        if col % 2:
            table[0, col] = -1 if col % 4 == 1 else 1 << 30
    got = kv.attend(cache, q, table, L, cu=cu, max_new=new, max_len=1000, window=window, sinks=sinks)
    check(got, want, tol)


@pytest.mark.parametrize("new", [1, 80])
def test_attend_pages_that_are_missing(dev, new):
    """A page that is needed and is not there makes the rows that need it NaN and no others."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, [new, new], [500, 400], 4, 4, 64, 64, BF)
    want, tol = R.attend(cache, q, table, L, cu)
    table[0, 2] = 1 << 30
    got = kv.attend(cache, q, table, L, cu=cu, max_new=new, max_len=500)
    assert torch.isnan(got[:new]).all()
    check(got[new:], want[new:], tol[new:])
    L[1] = 100 * 64  # past the table's width
    assert torch.isnan(kv.attend(cache, q, table, L, cu=cu, max_new=new, max_len=500)[new:]).all()


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("dtype,q_scale", [(BF, 1e30), (BF, 1e-30), (HF, 6e4), (HF, 1e-6), (BF, 0.0)])
def test_attend_query_range(dev, new, dtype, q_scale):
    """Queries near the types' borders: the scores stay finite because the keys are small."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, [new], [300], 4, 2, 128, 32, dtype, q_scale=1.0)
    x = q.float()
    q = (x / x.abs().max() * q_scale).to(dtype)
    if q_scale > 1:
        cache[2].mul_(4.0 / q_scale)
    want, tol = R.attend(cache, q, table, L, cu)
    check(kv.attend(cache, q, table, L, cu=cu, max_new=new), want, tol)


@pytest.mark.parametrize("new", [1, 100])
def test_attend_value_scales_far_apart(dev, new):
    """Pages of zeros (the smallest scale), one loud page, and the rest: no page's scale costs another's precision."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, [new], [1024], 4, 2, 64, 16, HF, q_scale=0.2)
    k, v, ks, vs = cache
    for i, p in enumerate(table[0].tolist()):
        if i % 3 == 0:
            v[p] = 0
            vs[p] = 1e-8 / 127
        if i == 7:
            vs[p] = 30.0
    want, tol = R.attend(cache, q, table, L, cu)
    check(kv.attend(cache, q, table, L, cu=cu, max_new=new), want, tol)
    vs.fill_(0.0)  # a cache whose values are all zero
    assert kv.attend(cache, q, table, L, cu=cu, max_new=new).abs().max().item() == 0.0


@pytest.mark.parametrize("new", [1, 100])
def test_attend_scores_far_below_zero(dev, new):
    """All scores of a row near -1e33: the softmax is that of their differences (here: of one key each)."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, [new], [130], 2, 1, 64, 16, BF)
    cache[0].copy_(cache[0].abs().clamp(min=1))
    q = -q.abs().clamp(min=0.5)
    cache[2].fill_(1e31)
    want, _ = R.attend(cache, q, table, L, cu)
    v = R.tokens(cache, table[0], 130)[1][:, 0]
    got = kv.attend(cache, q, table, L, cu=cu, max_new=new).double()
    # scores' fp32 roundings pick among keys whose scores are nearly the same: the output is some key's values
    near = (got[:, :, None] - v[None, None]).abs().amax(-1).amin(-1)
    assert (near <= 2.0 ** -8 * v.abs().max()).all() and (got - want).abs().amax(-1).le(2.0 ** -8 * v.abs().max()).float().mean() > 0.9


@pytest.mark.parametrize("new", [1, 64])
def test_attend_queries_that_are_not_numbers(dev, new):
    """An infinite or NaN query gives NaN in its own row and head, and nowhere else."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, [new, new], [90, 200], 4, 2, 64, 64, BF)
    want, tol = R.attend(cache, q, table, L, cu)
    q[0, 1, 3], q[new, 2, 5] = math.inf, math.nan
    got = kv.attend(cache, q, table, L, cu=cu, max_new=new)
    bad = torch.zeros(got.shape[:2], dtype=torch.bool, device=dev)
    bad[0, 1] = bad[new, 2] = True
    assert torch.isnan(got[bad]).all()
    check(got[~bad], want[~bad], tol[~bad])


@pytest.mark.parametrize("new", [1, 70])
def test_attend_strides_and_scale(dev, new):
    """q as a slice of wider rows, the table as a slice, lens as a column, another scale; a misaligned q is copied."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, [new, new], [100, 260], 6, 2, 64, 16, BF)
    want, tol = R.attend(cache, q, table, L, cu, scale=0.3)
    wide = torch.zeros((2 * new, 10, 64), dtype=BF, device=dev)
    wide[:, 1:7] = q
    tw = torch.full((2, table.shape[1] + 5), 1 << 30, dtype=torch.int32, device=dev)
    tw[:, 2:2 + table.shape[1]] = table
    lw = torch.zeros((2, 3), dtype=torch.int32, device=dev)
    lw[:, 1] = L
    args = dict(cu=cu, max_new=new, max_len=260, scale=0.3)
    check(kv.attend(cache, wide[:, 1:7], tw[:, 2:2 + table.shape[1]], lw[:, 1], **args), want, tol)
    flat = torch.zeros(q.numel() + 8, dtype=BF, device=dev)
    flat[3:3 + q.numel()] = q.flatten()
    check(kv.attend(cache, flat[3:3 + q.numel()].view(q.shape), table, L, **args), want, tol)
    check(kv.attend(cache, q.transpose(0, 1).contiguous().transpose(0, 1), table, L, **args), want, tol)
    if new == 1:
        check(kv.attend(cache, q, table.t().contiguous().t(), L, **args), want, tol)


HEAVY = [s for s in SHAPES if max(s[0]) * s[2] // s[3] > 16]


@pytest.mark.parametrize("new,lens,H,Hkv,hd,page,dtype", HEAVY)
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 4), (1000, 70)])
def test_attend_forms_for_much_work(dev, new, lens, H, Hkv, hd, page, dtype, window, sinks):
    """The kernels that calls with much work take (a bound of the lengths that is far off takes them here): two row
    tiles to a wave for heads of 64 and less, 128 rows to a workgroup; with and without splits of the keys."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, new, lens, H, Hkv, hd, page, dtype, seed=len(new) + H)
    want, tol = R.attend(cache, q, table, L, cu, window, sinks)
    for bound in (1 << 16, 1 << 22):
        check(kv.attend(cache, q, table, L, cu=cu, max_new=max(new), max_len=bound, window=window, sinks=sinks), want, tol)


@pytest.mark.parametrize("new,lens,dtype", [([2070, 2100], [2100, 2100], BF), ([4200], [5000], HF), ([1500, 1400, 1301], [1500, 1463, 2000], BF)])
def test_attend_eight_waves(dev, new, lens, dtype):
    """Enough rows for 256 to a workgroup on every CU, the last tiles of a sequence partly filled."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, new, lens, 16, 16, 128, 32, dtype, seed=len(new))
    want, tol = R.attend(cache, q, table, L, cu)
    check(kv.attend(cache, q, table, L, cu=cu, max_new=max(new), max_len=max(lens)), want, tol)


@pytest.mark.parametrize("new,lens,H,Hkv,window,sinks", [([300], [3001], 4, 1, 0, 0), ([300], [3001], 4, 1, 1000, 70), ([300, 1, 257], [900, 1000, 4000], 16, 4, 0, 0),
                                                         ([140, 129], [140, 5000], 14, 2, 2048, 5), ([2070, 2100], [2100, 5000], 16, 16, 2048, 4)])
def test_attend_eight_waves_over_a_context(dev, new, lens, H, Hkv, window, sinks):
    """256 rows to a workgroup where most keys are earlier ones, with and without windows, and in split parts."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, new, lens, H, Hkv, 128, 64, BF, seed=len(new) + H)
    want, tol = R.attend(cache, q, table, L, cu, window, sinks)
    check(kv.attend(cache, q, table, L, cu=cu, max_new=max(new), max_len=max(lens), window=window, sinks=sinks), want, tol)
    check(kv.attend(cache, q, table, L, cu=cu, max_new=max(new), max_len=1 << 16, window=window, sinks=sinks), want, tol, "high bound")


def test_short_and_long_way_agree(dev, monkeypatch):
    """The native way for arguments of the usual form and the one that looks at any: the same bits."""
    from uwc_amd import _lib, kv
    cache, qkv, table, c, cos, sin, cu, w = append_problem(dev, [70, 3], [5, 40], 4, 2, 64, 16, HF, True)
    other = [x.clone() for x in cache]

    def run(cache):
        q = kv.append(cache, qkv, table, c, cos, sin, cu=cu, q_norm=w[0], k_norm=w[1])
        n = c + (cu[1:] - cu[:-1])
        return (q, kv.attend(cache, q, table, n, cu=cu, window=20, sinks=2), kv.attend(cache, q, table, n, cu=cu, max_new=70, scale=0.2),
                *kv.read(cache, table, c, cu, 73, dtype=HF), *cache)

    short = run(cache)

    class Never:
        append = attend = read = staticmethod(lambda *a: None)

    monkeypatch.setattr(_lib, "_KV", Never)
    for a, b in zip(short, run(other)):
        assert torch.equal(a, b)


def test_refusals_of_the_library_reach_the_caller(dev):
    from uwc_amd import _lib, kv
    cache, q, table, L, cu = problem(dev, [1], [20], 4, 2, 64, 16, BF)
    with pytest.raises(_lib.UwcError, match="scale of the scores must be positive"):
        kv.attend(cache, q, table, L, scale=0.0)


def test_offsets_past_32_bits(dev):
    """Pages beyond 2^31 bytes of keys: appended to, attended over, read back."""
    from uwc_amd import kv
    pages, Hkv, hd, page = 17000, 8, 128, 128
    k = torch.empty((pages, Hkv, page, hd), dtype=torch.int8, device=dev)
    v = torch.empty((pages, Hkv, hd, page), dtype=torch.int8, device=dev)
    cache = (k, v, torch.ones((pages, Hkv), device=dev), torch.ones((pages, Hkv), device=dev))
    ids = [16999, 3, 16500, 16800]
    g = torch.Generator().manual_seed(5)
    small = R.make_cache(4, Hkv, hd, page, g, dev)
    for i, p in enumerate(ids):
        for big, part in zip(cache, small):
            big[p] = part[i]
    table, near = R.ints([ids], dev), R.ints([[0, 1, 2, 3]], dev)
    qkv = torch.randn((1, (16 + 16) * hd), generator=g).to(BF).to(dev)
    ang = torch.rand((512, hd), generator=g).to(dev)
    args = (R.ints([450], dev), ang.cos(), ang.sin())
    q = kv.append(cache, qkv, table, *args)
    assert torch.equal(q, kv.append(small, qkv, near, *args))
    L = R.ints([451], dev)
    assert torch.equal(kv.attend(cache, q, table, L), kv.attend(small, q, near, L))
    span = (R.ints([100], dev), R.ints([0, 351], dev), 351)
    for a, b in zip(kv.read(cache, table, *span), kv.read(small, near, *span)):
        assert torch.equal(a, b)


APPENDS = [  # new, ctx, H, Hkv, hd, page, dtype, norm
    ([1], [0], 16, 8, 128, 64, BF, True),
    ([1, 1, 1, 1], [777, 64, 15, 1], 32, 8, 128, 32, BF, False),
    ([1, 1, 1], [31, 127, 16], 7, 1, 64, 16, HF, True),
    ([3, 0, 130, 1], [5, 9, 64, 127], 4, 2, 128, 128, BF, True),
    ([200, 77], [0, 50], 6, 2, 64, 64, HF, False),
    ([129, 128, 9], [3, 128, 120], 2, 2, 32, 128, BF, True),
    ([300, 1, 16], [33, 48, 15], 16, 8, 128, 16, HF, True),
    ([150, 40], [0, 1], 8, 4, 128, 64, BF, False),
    ([100], [61], 3, 1, 128, 32, HF, True),
]


def append_problem(dev, new, ctx, H, Hkv, hd, page, dtype, norm, seed=3, loud=1.0):
    g = torch.Generator().manual_seed(seed)
    lens = [n + c for n, c in zip(new, ctx)]
    table, pages = R.make_table(lens, page, g, dev)
    cache = R.make_cache(pages, Hkv, hd, page, g, dev)
    qkv = (loud * torch.randn((sum(new), (H + 2 * Hkv) * hd), generator=g)).to(dtype).to(dev)
    ang = (6 * torch.randn((max(lens) + 2, hd), generator=g)).to(dev)
    w = [(1 + 0.1 * torch.randn(hd, generator=g)).to(dev) if norm else None for _ in range(2)]
    return cache, qkv, table, R.ints(ctx, dev), ang.cos(), ang.sin(), R.cumulative(new, dev), w


@pytest.mark.parametrize("new,ctx,H,Hkv,hd,page,dtype,norm", APPENDS)
@pytest.mark.parametrize("loud", [1.0, 0.01])  # scales that mostly grow, scales that mostly stay
def test_append_matches_definition(dev, new, ctx, H, Hkv, hd, page, dtype, norm, loud):
    from uwc_amd import kv
    cache, qkv, table, c, cos, sin, cu, w = append_problem(dev, new, ctx, H, Hkv, hd, page, dtype, norm and loud == 1.0, loud=loud)
    before = [x.clone() for x in cache]
    q = kv.append(cache, qkv, table, c, cos, sin, cu=cu, q_norm=w[0], k_norm=w[1])
    x = qkv.double().view(len(qkv), -1, hd)
    touched = {}
    at = 0
    for b, (n, p0) in enumerate(zip(new, ctx)):
        rows, pos = x[at:at + n], slice(p0, p0 + n)
        parts = [R.norm_turn(rows[:, :H], w[0], cos[pos], sin[pos], 1e-6), R.norm_turn(rows[:, H:H + Hkv], w[1], cos[pos], sin[pos], 1e-6)]
        val, mag = parts[0]
        # norm: hd roundings of the sum of squares at most, halved by the root, and six more; the rotation: three
        fuzz = (hd / 2 + 12) * 2.0 ** -24
        half = torch.finfo(dtype).eps / 2
        check(q[at:at + n], val, half * val.abs() + 1.01 * fuzz * mag + 2.0 ** -25, "q")
        for side, (val, mag) in ((0, parts[1]), (1, (rows[:, H + Hkv:], torch.zeros_like(rows[:, H + Hkv:])))):
            data, scale, was, old = cache[side], cache[2 + side], before[side], before[2 + side]
            get = lambda t, page_id, slot: t[page_id, :, slot] if side == 0 else t[page_id, :, :, slot]
            for col in range(p0 // page, -(-(p0 + n) // page)) if n else ():
                pg = int(table[b, col])
                lo, hi = max(p0, col * page), min(p0 + n, (col + 1) * page)
                touched.setdefault(side, set()).add(pg)
                v = val[lo - p0:hi - p0]
                m = mag[lo - p0:hi - p0] * fuzz
                s = torch.clamp(v.abs().amax((0, 2)), min=1e-8) / 127
                slack = m.amax((0, 2)) / 127 + s * 2.0 ** -22
                held = lo > col * page
                if held:
                    s = torch.maximum(s, old[pg].double())
                assert ((scale[pg].double() - s).abs() <= slack).all(), "scale"
                s = scale[pg].double()
                for slot in range(lo - col * page, hi - col * page):
                    i = slot + col * page - lo
                    z = get(data, pg, slot).double()
                    assert ((z * s[:, None] - v[i]).abs() <= s[:, None] * (0.5 + 127 * 2.0 ** -22) + m[i]).all(), "new token"
                for slot in range(lo - col * page if held else 0):
                    z, z0 = get(data, pg, slot), get(was, pg, slot)
                    same = s == old[pg].double()
                    assert torch.equal(z[same], z0[same])
                    off = (z.double() * s[:, None] - z0.double() * old[pg].double()[:, None]).abs()
                    assert (off <= s[:, None] * (0.5 + 127 * 2.0 ** -22)).all(), "older token"
        at += n
    for side in (0, 1):  # other pages keep every byte
        rest = [i for i in range(cache[0].shape[0]) if i not in touched.get(side, set())]
        assert torch.equal(cache[side][rest], before[side][rest]) and torch.equal(cache[2 + side][rest], before[2 + side][rest])


def test_append_in_steps_equals_its_rounding(dev):
    """A prompt in one call and in chunks that end inside pages: fresh pages get the same bytes, and token by
    token every value stays within the roundings that its page's growing scale made."""
    from uwc_amd import kv
    H, Hkv, hd, page = 4, 2, 64, 16
    cache, qkv, table, _, cos, sin, _, w = append_problem(dev, [100], [0], H, Hkv, hd, page, BF, True)
    other = [x.clone() for x in cache]
    zero = R.ints([0], dev)
    q = kv.append(cache, qkv, table, zero, cos, sin, cu=R.ints([0, 100], dev), q_norm=w[0], k_norm=w[1])
    for lo, hi in ((0, 32), (32, 96), (96, 100)):
        part = kv.append(other, qkv[lo:hi], table, R.ints([lo], dev), cos, sin, cu=R.ints([0, hi - lo], dev), q_norm=w[0], k_norm=w[1])
        assert torch.equal(part, q[lo:hi])
    span = (table, zero, R.ints([0, 100], dev), 100)
    for a, b in zip(kv.read(cache, *span, dtype=HF), kv.read(other, *span, dtype=HF)):
        assert torch.equal(a, b)
    for t in range(100):
        part = kv.append(other, qkv[t:t + 1], table, R.ints([t], dev), cos, sin, q_norm=w[0], k_norm=w[1])
        assert torch.equal(part, q[t:t + 1])
    ids = table[0, :7].long()
    for side in (0, 1):
        assert torch.equal(cache[2 + side][ids], other[2 + side][ids])  # the page's maximum is the same
        s = cache[2 + side][ids].double()
        s = s.repeat_interleave(page, 0)[:100, :, None]
        a, b = R.tokens(cache, table[0], 100)[side], R.tokens(other, table[0], 100)[side]
        assert ((a - b).abs() <= s * 8.5).all()  # at most 15 growths of half a step of a smaller scale, and its own


def test_append_not_numbers_and_bad_places(dev):
    """A NaN or infinite head reaches its page's scale; rows without a page, or past the rotation tables, give
    NaN queries and write nothing; padding rows give zeros."""
    from uwc_amd import kv
    new, ctx = [1, 1, 1, 1], [40, 5, 20, 63]
    cache, qkv, table, c, cos, sin, _, _ = append_problem(dev, new, ctx, 4, 2, 64, 16, BF, False)
    qkv[0, 4 * 64 + 7] = math.nan    # k head 0
    qkv[1, 7 * 64 + 1] = math.inf    # v head 1
    table[2, 1] = 1 << 30
    before = [x.clone() for x in cache]
    q = kv.append(cache, qkv, table, c, cos[:63], sin[:63])
    assert torch.isnan(q[2]).all() and torch.isnan(q[3]).all() and not torch.isnan(q[:2]).any()
    p0, p1, p3 = (int(table[b, ctx[b] // 16]) for b in (0, 1, 3))
    assert torch.isnan(cache[2][p0, 0]) and not torch.isnan(cache[2][p0, 1]) and not torch.isnan(cache[3][p0]).any()
    assert torch.isinf(cache[3][p1, 1]) and torch.isfinite(cache[3][p1, 0]) and torch.isfinite(cache[2][p1]).all()
    assert torch.isnan(cache[2][p3]).all()  # a key whose position has no rotation
    rest = [i for i in range(cache[0].shape[0]) if i not in (p0, p1, p3)]
    for x, y in zip(cache, before):
        assert torch.equal(x[rest], y[rest])
    cu = R.ints([0, 1, 2, 2, 2], dev)
    assert not kv.append(cache, qkv, table, c, cos, sin, cu=cu)[2:].any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd,page,Hkv", [(128, 64, 8), (128, 16, 1), (64, 128, 3), (32, 32, 2)])
def test_read_is_the_rounded_product(dev, dtype, hd, page, Hkv):
    from uwc_amd import kv
    n, start = [1, 0, 65, 200], [129, 3, 0, 17]
    g = torch.Generator().manual_seed(1)
    table, pages = R.make_table([a + b for a, b in zip(n, start)], page, g, dev)
    k, v, ks, vs = cache = R.make_cache(pages, Hkv, hd, page, g, dev)
    ko, vo = kv.read(cache, table, R.ints(start, dev), R.cumulative(n, dev), sum(n), dtype=dtype)
    at = 0
    for b in range(len(n)):
        pos = torch.arange(start[b], start[b] + n[b], device=dev)
        pg, sl = table[b, pos // page].long(), pos % page
        assert torch.equal(ko[at:at + n[b]], (k[pg, :, sl].float() * ks[pg][..., None]).to(dtype))
        assert torch.equal(vo[at:at + n[b]], (v[pg, :, :, sl].float() * vs[pg][..., None]).to(dtype))
        at += n[b]
    table[3, 0] = -1
    ko, vo = kv.read(cache, table, R.ints(start, dev), R.cumulative(n, dev), sum(n), dtype=dtype)
    first = min(page - 17 if page > 17 else 0, 200)
    assert torch.isnan(ko[66:66 + first]).all() and torch.isnan(vo[66:66 + first]).all()
    assert not torch.isnan(ko[66 + first:]).any() and not torch.isnan(vo[66 + first:]).any()


def test_no_sequences(dev):
    """A padded batch without a sequence: zeros."""
    from uwc_amd import kv
    cache = kv.new_cache(2, 2, 64, 16, dev)
    table, none, cu = torch.zeros((0, 3), dtype=torch.int32, device=dev), R.ints([], dev), R.ints([0], dev)
    q = torch.ones((70, 4, 64), dtype=BF, device=dev)
    assert not kv.attend(cache, q, table, none, cu=cu).any()
    cos = torch.ones((4, 64), device=dev)
    assert not kv.append(cache, torch.ones((9, 8 * 64), dtype=BF, device=dev), table, none, cos, cos, cu=cu).any()


@pytest.mark.parametrize("new", [1, 5, 300])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_attend_lengths_past_the_table(dev, new, window, sinks):
    """Lengths that no table could hold end at once, in NaN; another sequence beside is as it was."""
    from uwc_amd import kv
    cache, q, table, L, cu = problem(dev, [new, new], [400, 400], 8, 2, 64, 16, BF)
    want, tol = R.attend(cache, q, table, L, cu, window if window < 1000 else 0, sinks if window < 1000 else 0)
    L[0] = 2 ** 31 - 100
    got = kv.attend(cache, q, table, L, cu=cu, max_new=new, max_len=400, window=window, sinks=sinks)
    assert torch.isnan(got[:new]).all()
    check(got[new:], want[new:], tol[new:])
    got = kv.attend(cache, q, table, L, cu=cu, max_new=new, max_len=1 << 22, window=window, sinks=sinks)
    assert torch.isnan(got[:new]).all()
    check(got[new:], want[new:], tol[new:])


def test_nothing_to_do(dev):
    from uwc_amd import kv
    cache = kv.new_cache(2, 2, 64, 16, dev)
    e = lambda *s: torch.empty(s, dtype=BF, device=dev)
    none, table = R.ints([], dev), torch.zeros((0, 1), dtype=torch.int32, device=dev)
    cos = torch.ones((4, 64), device=dev)
    assert kv.append(cache, e(0, 8 * 64), table, none, cos, cos).shape == (0, 4, 64)
    assert kv.attend(cache, e(0, 4, 64), table, none).shape == (0, 4, 64)
    assert kv.read(cache, table, none, R.ints([0], dev), 0)[0].shape == (0, 2, 64)
    zero = R.ints([0], dev)
    t1 = R.ints([[0]], dev)
    q = kv.append(cache, torch.ones((1, 8 * 64), dtype=BF, device=dev), t1, zero, cos, 0 * cos)
    assert (q == 1).all()
    q = kv.append(cache, torch.ones((1, 4 * 64), dtype=BF, device=dev), t1, zero, cos, 0 * cos)  # no q heads
    assert q.shape == (1, 0, 64)


def test_graph_replays(dev):
    """A decode step captured once and replayed while the sequences grow, against the eager step."""
    from uwc_amd import kv
    H, Hkv, hd, page, B = 8, 2, 64, 16, 3
    ctx0 = [700, 15, 3]
    cache, _, table, c, cos, sin, _, w = append_problem(dev, [8] * B, ctx0, H, Hkv, hd, page, BF, True)
    eager = [x.clone() for x in cache]
    g = torch.Generator().manual_seed(9)
    rows = torch.randn((6, B, (H + 2 * Hkv) * hd), generator=g).to(BF).to(dev)
    qkv, lens = rows[0].clone(), c + 1

    def step(cache):
        q = kv.append(cache, qkv, table, c, cos, sin, q_norm=w[0], k_norm=w[1])
        return kv.attend(cache, q, table, lens, max_len=720)

    spare = [x.clone() for x in cache]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # on another stream than the tensors' own
        step(spare)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for t in range(6):
        qkv.copy_(rows[t])
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want), t
        for x, y in zip(cache, eager):
            assert torch.equal(x, y), t
        c += 1
        lens += 1
