"""Paged key / value cache: pages and slots of a step, rows written into them, attention over them. Whole numbers against a plain loop, attention against softmax in 64 bits."""
import pytest
import torch

import paged_cases as ref
from helpers import check_status

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _dev(x):
    return torch.tensor(x, dtype=I32, device="cuda")


# ---- pages ----------------------------------------------------------------------------------------------------------------
def _requests(seed, B, page, most_cached, most_new, spare, ended=0.0, idle=0.2):
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi: torch.randint(lo, hi, (B,), generator=g).tolist()
    cached, new = r(0, most_cached + 1), r(1, most_new + 1)
    kind = torch.rand(B, generator=g)
    new = [-1 if kind[b] < ended else 0 if kind[b] < ended + idle else new[b] for b in range(B)]
    width = -(-(most_cached + most_new) // page)
    held = [-(-c // page) for c in cached]
    n_pages = sum(held) + spare
    ids = torch.randperm(n_pages, generator=g).tolist()
    table, at = [[-7] * width for _ in range(B)], 0
    for b in range(B):
        for j in range(held[b]):
            table[b][j] = ids[at]
            at += 1
    free = ids[at:] + [-9] * at
    return cached, new, table, free, n_pages - at


def _check_plan(cached, new, table, free, n_free, page, max_rows, pitch=0, in_place=False, ld=None):
    import plz_ops as ops
    width = len(table[0])
    tab = torch.full((len(table), ld or width), -5, dtype=I32, device="cuda")[:, :width]
    tab.copy_(_dev(table))
    L, F, nf = _dev(cached), _dev(free), _dev([n_free])
    p = ops.plan_pages(L, _dev(new), tab, F, nf, page, max_rows, pitch, **({"lengths_out": L, "n_free_out": nf} if in_place else {}))
    want = ref.plan(cached, new, table, free, n_free, page, max_rows, pitch)
    got = (p.lengths, p.n_free, p.starts, p.slots, p.positions, p.status)
    for name, a, b in zip(("lengths", "n_free", "starts", "slots", "positions", "status"), got, want):
        assert a.tolist() == ([b] if name == "n_free" else b), name
    assert tab.tolist() == table and F.tolist() == free
    if in_place:
        assert p.lengths.data_ptr() == L.data_ptr()
    else:
        assert L.tolist() == cached and nf.tolist() == [n_free]
    return want[5]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,page,most_cached,most_new", [(1, 16, 0, 1), (3, 1, 20, 5), (64, 16, 300, 1), (37, 24, 100, 700), (300, 64, 1000, 40), (1000, 8, 50, 30)])
def test_plan(B, page, most_cached, most_new, in_place):
    a = _requests(B + page, B, page, most_cached, most_new, spare=B * (most_new // page + 2), ended=0.1)
    rows = sum(max(n, 0) for n in a[1])
    _check_plan(*a, page, rows + 11, in_place=in_place, ld=len(a[2][0]) + 3)


def test_plan_without_enough_pages_or_rows():
    """Statuses 1 and 2: few free pages, a table that is too narrow for some, rows past the step's."""
    seen = []
    for seed in range(6):
        cached, new, table, free, n_free = _requests(seed, 40, 8, 60, 50, spare=60, ended=0.1)
        table = [t[:10] for t in table]
        cached = [min(c, 80) for c in cached]
        cached[seed] = -3
        seen.append(set(_check_plan(cached, new, table, free, n_free, 8, sum(max(n, 0) for n in new) - 20 * seed)))
    assert all({0, 2} <= s for s in seen) and sum(1 in s for s in seen) >= 3


@pytest.mark.parametrize("pitch", [1, 4, 7])
def test_plan_of_a_padded_batch(pitch):
    a = _requests(pitch, 50, 16, 200, 5, spare=100, ended=0.1, idle=0.3)
    _check_plan(*a, 16, 50 * pitch + 5, pitch=pitch)


def test_plan_with_fewer_tokens_a_request_than_its_pages_hold():
    import plz_ops as ops
    cached, new = [5, 9, 10, 0, 11, 8, 10], [5, 2, 0, 11, -1, 2, -1]
    table = torch.full((7, 3), -1, dtype=I32, device="cuda")
    for b, n in enumerate(cached):
        table[b, : -(-n // 4)] = _dev([b * 3 + j for j in range(-(-n // 4))])
    want = [0, 2, 0, 2, 2, 0, 0]
    for B in (7, 1000):                      # the small kernel and the large one
        more = B - 7
        p = ops.plan_pages(_dev(cached + [0] * more), _dev(new + [0] * more), torch.cat([table.clone(), torch.full((more, 3), -1, dtype=I32, device="cuda")]), _dev(list(range(30, 60))), _dev([30]),
                           4, 30, max_tokens=10)
        assert p.status.tolist() == want + [0] * more
        assert p.lengths.tolist() == [10, 9, 10, 0, 11, 10, 0] + [0] * more


def test_plan_of_nothing():
    import plz_ops as ops
    e = torch.zeros(0, dtype=I32, device="cuda")
    p = ops.plan_pages(e, e, e.view(0, 4), _dev([3, 4]), _dev([2]), 16, 5)
    assert p.slots.tolist() == p.positions.tolist() == [-1] * 5 and p.starts.tolist() == [0] and p.n_free.tolist() == [2]
    p = ops.plan_pages(_dev([0]), _dev([3]), e.view(1, 0), e, _dev([0]), 16, 3)       # no pages, no table
    assert p.status.tolist() == [2] and p.lengths.tolist() == [0]
    p = ops.plan_pages(_dev([0]), _dev([3]), _dev([[0]]), e, _dev([5]), 16, 3)        # a count of free pages that the stack does not hold
    assert p.status.tolist() == [1] and p.n_free.tolist() == [0]


def test_plan_of_more_requests_than_threads_and_of_the_most():
    B = 16384
    a = ([5] * B, [1] * B, [[b, -1] for b in range(B)], [B + i for i in range(B // 2)] + [-1] * B, B // 2)
    _check_plan(*a, 5, B)


def test_planned_steps_captured():
    """A captured step in place, replayed: lengths grow, pages come, requests end, the pages that they give back serve later ones."""
    import plz_ops as ops
    B, page, width, n_pages, rows = 6, 4, 5, 14, 12
    L, new, tab, F, nf = _dev([0] * B), _dev([0] * B), _dev([[-1] * width] * B), _dev(list(range(n_pages))), _dev([n_pages])
    state = ([0] * B, [[-1] * width for _ in range(B)], list(range(n_pages)), n_pages)
    step = lambda: ops.plan_pages(L, new, tab, F, nf, page, rows, lengths_out=L, n_free_out=nf)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = step()
    g = torch.Generator().manual_seed(1)
    for i in range(30):
        n = torch.randint(-1, 4, (B,), generator=g).tolist()
        new.copy_(_dev(n))
        graph.replay()
        cached, table, free, n_free = state
        lengths, left, starts, slots, positions, status = ref.plan(cached, n, table, free, n_free, page, rows)
        assert (p.lengths.tolist(), p.n_free.tolist(), p.slots.tolist(), p.status.tolist()) == (lengths, [left], slots, status), i
        assert tab.tolist() == table and F.tolist()[:left] == free[:left]
        state = (lengths, table, free, left)


# ---- rows -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,width,page,dtype", [(1, 8, 1, torch.bfloat16), (7, 40, 16, torch.bfloat16), (64, 1024, 16, torch.bfloat16), (100, 24, 5, torch.float32), (9000, 128, 64, torch.bfloat16), (9001, 1024, 16, torch.bfloat16),
                                                   (3001, 520, 24, torch.float32), (33, 4096, 8, torch.uint8)])
@pytest.mark.parametrize("strided", [False, True])
def test_write(rows, width, page, dtype, strided):
    import plz_ops as ops
    g = torch.Generator(device="cuda").manual_seed(rows)
    rnd = lambda *s: torch.randint(0, 250, s, generator=g, device="cuda").to(dtype)
    pages = rows // page + 3
    unit = 16 // dtype.itemsize
    k, v = (rnd(rows, width + unit)[:, :width] if strided else rnd(rows, width) for _ in range(2))
    kp, vp = (rnd(pages, 2, page, width + 2 * unit)[:, 1, :, :width] if strided else rnd(pages, page, width) for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows].to(I32)
    slots[torch.rand(rows, generator=g, device="cuda") < 0.2] = -1
    slots[-1] = pages * page                      # past the pool
    want = [t.clone() for t in (kp, vp)]
    good = (slots >= 0) & (slots < pages * page)
    for t, x in zip(want, (k, v)):
        t.view(-1, width)[slots[good].long()] = x[good]
    whole = [t._base.clone() if t._base is not None else None for t in (kp, vp)]
    ops.write_pages(k, v, slots, kp, vp)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    for t, before in zip((kp, vp), whole):
        if before is not None and strided:
            b = before.view(pages, 2, page, -1)
            b[:, 1, :, :width] = t
            assert torch.equal(t._base.view(pages, 2, page, -1), b)      # nothing else was touched
    ops.write_pages(k[:0], v[:0], slots[:0], kp, vp)


# ---- attention --------------------------------------------------------------------------------------------------------------
def _case(seed, lengths, hq, hk, d, page, spare=3, fill=float("nan"), wide=2):
    """Requests of these lengths over shuffled pages; rows that belong to nobody hold `fill`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, width = len(lengths), max(-(-max(lengths) // page), 1) + wide
    need = [-(-n // page) for n in lengths]
    n_pages = sum(need) + spare
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(I32)
    table = torch.full((B, width), -1, dtype=I32, device="cuda")
    kp, vp = (torch.full((n_pages, page, hk * d), fill, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = 0
    for b, n in enumerate(lengths):
        table[b, : need[b]] = ids[at: at + need[b]]
        for t in (kp, vp):
            rows = torch.randn(n, hk * d, generator=g, device="cuda").bfloat16()
            pool = t.view(-1, hk * d)
            pos = torch.arange(n, device="cuda")
            if n:
                pool[table[b, pos // page].long() * page + pos % page] = rows
        at += need[b]
    q = torch.randn(B, hq * d, generator=g, device="cuda").bfloat16()
    return q, kp, vp, table, _dev(lengths)


def _close(got, want, err):
    want, err, got = want.cpu(), err.cpu(), got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    off = (got - want).abs() - (2.0 ** -8 * want.abs() + err)
    assert (off[~want.isnan()] <= 0).all(), float(off.nan_to_num().max())


RAGGED = [0, 1, 15, 16, 17, 0, 300, 31, 33, 1000, 64, 2, 0]


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (1, 1, 128), (7, 1, 128), (8, 1, 64), (12, 2, 64), (20, 4, 128), (32, 2, 128), (9, 1, 64), (40, 2, 128), (17, 1, 256), (8, 2, 256), (16, 16, 64)])
@pytest.mark.parametrize("page", [16, 24])
def test_attention_heads(hq, hk, d, page):
    import plz_ops as ops
    a = _case(hq * d + page, RAGGED, hq, hk, d, page)
    got = ops.attention_decode_paged(*a, hq, hk, d)
    check_status()
    _close(got, *ref.attention(*a, hq, hk, d))
    assert (got[0] == 0).all() and (got[5] == 0).all()


@pytest.mark.parametrize("page", [1, 5, 8, 64, 128])
@pytest.mark.parametrize("lengths", [[1], [0], [2049], [4097, 3], [5] * 300, [16, 0] * 200, [3000, 1, 1, 1], list(range(0, 130))], ids=str)
def test_attention_lengths(page, lengths):
    import plz_ops as ops
    a = _case(page + len(lengths), lengths, 8, 2, 128, page)
    _close(ops.attention_decode_paged(*a, 8, 2), *ref.attention(*a, 8, 2, 128))
    check_status()


@pytest.mark.parametrize("hq,hk,d,page,B,T", [(32, 8, 128, 16, 70, 1500), (16, 16, 64, 64, 200, 700), (8, 2, 256, 32, 40, 3000), (40, 2, 128, 16, 60, 5000), (4, 1, 128, 16, 1, 600000), (9, 3, 64, 128, 2000, 300)])
def test_attention_with_many_steps(hq, hk, d, page, B, T):
    """Enough work for many steps in every warp: right, and the same bits each time."""
    import plz_ops as ops
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(T // 2, T + 1, (B,), generator=g).tolist()
    lengths[B // 3] = 0 if B > 1 else lengths[0]
    width = -(-T // page)
    dev = torch.Generator(device="cuda").manual_seed(B)
    table = torch.randperm(B * width, generator=dev, device="cuda").to(I32).view(B, width)
    kp, vp = (torch.randn(B * width, page, hk * d, generator=dev, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(B, hq * d, generator=dev, device="cuda").bfloat16()
    a = (q, kp, vp, table, _dev(lengths))
    got = [ops.attention_decode_paged(*a, hq, hk, d) for _ in range(4)]
    check_status()
    _close(got[0], *ref.attention(*a, hq, hk, d))
    assert all(torch.equal(got[0], x) for x in got[1:])


@pytest.mark.parametrize("hq,hk,d,page,lengths", [(4, 1, 128, 16, [400003]), (8, 2, 64, 24, [250001, 17, 130000]), (4, 1, 256, 64, [120007]), (12, 1, 128, 16, [90001, 300007])])
def test_long_requests_have_every_step_in_them(hq, hk, d, page, lengths):
    """Column c of a value is 1 in the c-th of d equal stretches of its request and 0 elsewhere, so result c is the weight of that stretch, about 1 / d: one step (16 tokens, 32 of 64-wide heads) more or
    less changes it by 16 d / T of itself (32 d / T), 5e-3 or more here. Its rounding to bf16 is half of finfo.eps = 2^-7 of itself at most, 2^-8 = 3.9e-3. Head 0 weighs all tokens alike, the others by random scores. Other errors, by T tokens cut in stretches of
    n = T Hkv / 16 / SMs / 4 + 1 steps or fewer: a weight 2 (d + 4) 2^-23 sum |q k| + 2^-21, a sum of weights or products 2^-23 for each of a lane's 16 n terms and of 400 parts."""
    import plz_ops as ops
    g = torch.Generator(device="cuda").manual_seed(d + page)
    B, width = len(lengths), -(-max(lengths) // page)
    table = torch.randperm(B * width, generator=g, device="cuda").to(I32).view(B, width)
    kp, vp = (torch.full((B * width, page, hk * d), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = (torch.randn(B, hk, hq // hk, d, generator=g, device="cuda") / 2).bfloat16()
    q[:, :, 0] = 0
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    steps = sum(lengths) * hk // 16 // sms // 4 + 1
    cases = []
    for b, n in enumerate(lengths):
        pos = torch.arange(n, device="cuda")
        at = table[b, pos // page].long() * page + pos % page
        k = torch.randn(n, hk * d, generator=g, device="cuda").bfloat16()
        part = (pos * d // n)
        kp.view(-1, hk * d)[at] = k
        vp.view(-1, hk * d)[at] = torch.nn.functional.one_hot(part, d).repeat(1, hk).bfloat16()
        cases.append((n, part, k.view(n, hk, d)))
    got = ops.attention_decode_paged(q.view(B, -1), kp, vp, table, _dev(lengths), hq, hk, d).double().view(B, hk, hq // hk, d)
    check_status()

    def weights(w, part):                       # per head the share of every stretch
        return torch.zeros(hk, hq // hk, d, dtype=torch.float64, device="cuda").index_add_(2, part, w / w.sum(-1, keepdim=True))
    for b, (n, part, k) in enumerate(cases):
        s = torch.einsum("hgd,nhd->hgn", q[b].double(), k.double()) * d ** -0.5
        w = (s - s.amax(-1, keepdim=True)).exp()
        want = weights(w, part)
        size = torch.einsum("hgd,nhd->hgn", q[b].double().abs(), k.double().abs()).amax(-1, keepdim=True) * d ** -0.5
        rel = 2.0 ** -8 * (1 + 2.0 ** -8) + 2 * (2 * (d + 4) * 2.0 ** -23 * size + 2.0 ** -21 + (16 * min(steps, -(-n // 16)) + 400) * 2.0 ** -23)
        right = lambda x: bool(((x - want).abs() <= rel * want).all())
        assert right(got[b]), (b, float(((got[b] - want).abs() / (rel * want)).nan_to_num().max()))
        # what the bound has to notice: nothing, half of the request, and where all tokens weigh alike one step left out
        if n > 1000:
            half, step = w.clone(), w.clone()
            half[..., n // 2:] = 0
            tok = 32 if d == 64 else 16
            step[..., n // 3 // tok * tok:][..., :tok] = 0
            assert not any(right(x) for x in (torch.zeros_like(want), weights(half, part), weights(step, part)))


@pytest.mark.parametrize("hq,hk,d", [(8, 1, 128), (12, 1, 128), (8, 1, 64), (8, 1, 256), (12, 1, 64), (12, 1, 256)])
def test_long_sums_do_not_drift(hq, hk, d):
    """Ten thousand steps a warp, over pages that come again and again: sums that are rounded to nearest are off by about sqrt(n) 2^-25 of themselves after n steps, 6 times that or less, and weights by
    2^-21 (exponential and exponent); an error e moves a value over a border between two bf16 numbers, 2^-8 apart or more, in 2 e 2^8 of all cases or fewer. Sums that are cut instead lose n 2^-24."""
    import plz_ops as ops
    tok, warps = (32 if d == 64 else 16), (4 if d == 256 else 8) * torch.cuda.get_device_properties(0).multi_processor_count
    B, n_pages, page, n = 8, 256, 64, 10000
    width = n * warps * tok // page // B // hk
    g = torch.Generator(device="cuda").manual_seed(d)
    table = torch.randint(0, n_pages, (B, width), generator=g, device="cuda").int()
    kp = torch.randn(n_pages, page, hk * d, generator=g, device="cuda").bfloat16()
    vp = (1 + torch.rand(n_pages, page, hk * d, generator=g, device="cuda")).bfloat16()
    q = torch.randn(B, hq * d, generator=g, device="cuda").bfloat16()
    got = ops.attention_decode_paged(q, kp, vp, table, torch.full((B,), width * page, dtype=I32, device="cuda"), hq, hk, d).view(B, hk, hq // hk, d)
    check_status()
    often = torch.stack([torch.bincount(table[b], minlength=n_pages) for b in range(B)]).repeat_interleave(page, 1).double()
    k, v = (t.view(-1, hk, d).double().transpose(0, 1) for t in (kp, vp))
    s = q.view(B, hk, hq // hk, d).double() @ k.transpose(1, 2) * d ** -0.5
    w = (s - s.amax(-1, keepdim=True)).exp() * often[:, None, None]
    want = (w / w.sum(-1, keepdim=True)) @ v
    e = 6 * n ** 0.5 * 2.0 ** -25 + 2.0 ** -21
    assert float((got.double() != want.bfloat16().double()).double().mean()) <= 2 * e * 2 ** 8


@pytest.mark.parametrize("hq,hk,d", [(8, 1, 64), (3, 1, 128), (12, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("shape", ["rising", "falling", "saw", "back and forth"])
def test_references_that_move_over_many_steps(hq, hk, d, shape):
    """Scores between -40 and 0 that go up or down again and again within a warp's 150 steps, so that sums of earlier steps count for nothing, for everything or in part. Columns are the parts of the period.
    A weight is off by 2 ((d + 4) 2^-23 40 + 2^-21), a sum of positive products by 2^-23 for each of a warp's 16 * 150 tokens and 2400 parts, and bf16 by 2^-8, all of itself."""
    import plz_ops as ops
    tok, warps = (32 if d == 64 else 16), (4 if d == 256 else 8) * torch.cuda.get_device_properties(0).multi_processor_count
    page, period = 64, 100 * tok + 37
    n = 150 * warps * tok // page * page + 5
    pos = torch.arange(n, device="cuda")
    x = (pos % period).double() / period
    s = {"rising": 40 * (pos.double() / n - 1), "falling": -40 * pos.double() / n, "saw": -40 * x, "back and forth": -80 * (x - 0.5).abs()}[shape].bfloat16()
    part = pos * d // n if shape in ("rising", "falling") else pos % period * d // period
    pages = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(d)
    table = torch.randperm(pages, generator=g, device="cuda").to(I32)[None]
    at = table[0, pos // page].long() * page + pos % page
    kp, vp = (torch.zeros(pages, page, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kp.view(-1, d)[at, 0] = s
    vp.view(-1, d)[at, part] = 1.0
    q = torch.zeros(1, hq, d, dtype=torch.bfloat16, device="cuda")
    q[0, :, 0] = torch.tensor([1.0, 0.5, 0.25], device="cuda").repeat(4)[:hq]
    got = ops.attention_decode_paged(q.view(1, -1), kp, vp, table, _dev([n]), hq, hk, d, scale=1.0).view(hq, d).double()
    check_status()
    w = (s.double() * q[0, :, :1].double()).exp()
    want = torch.zeros(hq, d, dtype=torch.float64, device="cuda").index_add_(1, part, w / w.sum(1, keepdim=True))
    rel = 2.0 ** -8 * (1 + 2.0 ** -8) + 2 * (2 * ((d + 4) * 2.0 ** -23 * 40 + 2.0 ** -21) + (16 * 150 + 2400) * 2.0 ** -23)
    assert ((got - want).abs() <= rel * want + 2.0 ** -126).all(), float(((got - want).abs() / (rel * want)).nan_to_num().max())


@pytest.mark.parametrize("B", [2, 31, 32, 33, 64])
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (20, 1, 64), (4, 4, 256)])
@pytest.mark.parametrize("holes", ["none", "ends", "inside", "most"])
def test_attention_around_a_warp_of_requests(B, hq, hk, d, holes):
    """Up to 32 requests a warp holds every length itself, above the CTA shares them; requests without tokens first, last and in runs."""
    import plz_ops as ops
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(1, 400, (B,), generator=g)
    if holes == "ends":
        lengths[:B // 3] = lengths[B - B // 3:] = 0
    elif holes == "inside":
        lengths[1:B - 1] = 0
    elif holes == "most":
        lengths[torch.rand(B, generator=g) < 0.8] = 0
    a = _case(B * d, lengths.tolist(), hq, hk, d, 16)
    got = ops.attention_decode_paged(*a, hq, hk, d)
    check_status()
    _close(got, *ref.attention(*a, hq, hk, d))
    assert (got[lengths == 0] == 0).all()


@pytest.mark.parametrize("scale", [1.0, 0.02, -0.3, 0.0])
def test_attention_scale_and_layouts(scale):
    """Pitched q, out and table, pools that are slices of a larger one."""
    import plz_ops as ops
    q, kp, vp, table, L = _case(7, RAGGED, 8, 2, 64, 16)
    both = torch.full((kp.shape[0], 3, 16, 2 * 64 + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    k2, v2 = both[:, 0, :, 8:136], both[:, 2, :, 8:136]
    k2.copy_(kp), v2.copy_(vp)
    q2 = torch.full((len(RAGGED), 600), float("nan"), dtype=torch.bfloat16, device="cuda")[:, 8:520]
    q2.copy_(q)
    t2 = torch.full((len(RAGGED), table.shape[1] + 5), 1 << 30, dtype=I32, device="cuda")[:, 3:3 + table.shape[1]]
    t2.copy_(table)
    out = torch.full((len(RAGGED) + 1, 560), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.attention_decode_paged(q2, k2, v2, t2, L, 8, 2, 64, scale=scale, out=out[:-1, 16:528])
    _close(out[:-1, 16:528], *ref.attention(q, kp, vp, table, L, 8, 2, 64, scale))
    assert (out[-1] == 7).all() and (out[:, :16] == 7).all() and (out[:, 528:] == 7).all()


@pytest.mark.parametrize("growth", [0.0, 0.02, 0.5, -0.5])
def test_scores_that_grow_along_the_sequence(growth):
    import plz_ops as ops
    q, kp, vp, table, L = _case(11, [700, 90, 1], 8, 2, 128, 16)
    q[:, ::128] = 4.0
    for b, n in enumerate([700, 90, 1]):
        pos = torch.arange(n, device="cuda")
        pool = kp.view(-1, 256)
        at = table[b, pos // 16].long() * 16 + pos % 16
        pool[at, 0] = (growth * pos).bfloat16()
        pool[at, 128] = (growth * pos).bfloat16()
    _close(ops.attention_decode_paged(q, kp, vp, table, L, 8, 2), *ref.attention(q, kp, vp, table, L, 8, 2, 128))


def test_infinite_scores_are_what_a_softmax_makes_of_them():
    """All scores of a request -inf, or one of them +inf: no number; the others are untouched."""
    import plz_ops as ops
    q, kp, vp, table, L = _case(5, [40, 40, 40], 4, 1, 64, 8)
    q[:, ::64] = 1.0
    pos = torch.arange(40, device="cuda")
    at = [table[b, pos // 8].long() * 8 + pos % 8 for b in range(3)]
    kp.view(-1, 64)[at[0], 0] = float("-inf")
    kp.view(-1, 64)[at[2][17], 0] = float("inf")
    got = ops.attention_decode_paged(q, kp, vp, table, L, 4, 1, 64)
    assert got[0].isnan().all() and got[2].isnan().all()
    _close(got[1:2], *(t[1:2] for t in ref.attention(q, kp, vp, table, L, 4, 1, 64)))


def test_pages_and_lengths_that_do_not_exist():
    import plz_ops as ops
    lengths = [100, 50, 20, 300]
    q, kp, vp, table, L = _case(3, lengths, 8, 2, 128, 16, wide=0)
    bad = torch.zeros(1, dtype=I32, device="cuda")
    ops.attention_decode_paged(q, kp, vp, table, L, 8, 2, bad=bad)
    assert bad.item() == 0
    table[0, 2], table[1, 0], table[3, 5] = -1, kp.shape[0], 2 ** 31 - 1
    got = ops.attention_decode_paged(q, kp, vp, table, L, 8, 2, bad=bad)
    assert bad.item() == 1
    _close(got, *ref.attention(q, kp, vp, table, L, 8, 2, 128))
    bad.zero_()
    q, kp, vp, table, L = _case(3, lengths, 8, 2, 128, 16, wide=0, fill=0.5)
    for n in (2 ** 31 - 1, -5):
        L[3] = n
        _close(ops.attention_decode_paged(q, kp, vp, table, L, 8, 2, bad=bad), *ref.attention(q, kp, vp, table, L, 8, 2, 128))
        assert bad.item() == 1
        bad.zero_()
    table[2] = -1                                  # a request whose every page is missing: no weight at all
    L[3] = 300
    got = ops.attention_decode_paged(q, kp, vp, table, L, 8, 2)
    assert got[2].isnan().all()


@pytest.mark.parametrize("hq,hk,d", [(8, 1, 128), (4, 2, 64), (4, 1, 256), (9, 1, 128), (16, 1, 64), (17, 1, 256)])
def test_weights_enter_the_product_with_all_their_bits(hq, hk, d):
    """A weight w = e^s against tokens of weight 1 whose values are -w in three bf16 terms: what is left is the weight's own error. Off by 2^-23 w through the exponent (two roundings of 2^-24 of
    |s| log2(e) <= 1.45, times ln 2), 2^-22 w through the exponential, and by four sums below 2 that may drop 2^-24 of it each (all other products are multiples of 2^-24): 2^-21 in all. Two bf16 terms
    of w would leave up to 2^-18."""
    import plz_ops as ops
    s = -torch.arange(1, 201).double().div(256).bfloat16().double()      # scores, exact in bf16
    w, B = s.exp(), s.numel()
    terms, left = [], w.clone()
    for _ in range(3):
        terms.append(left.bfloat16().double())
        left = left - terms[-1]
    kp, vp = (torch.zeros(B, 4, hk * d, dtype=torch.float64) for _ in range(2))
    kp[:, 0, ::d] = s[:, None]
    vp[:, 0] = 1.0
    for i, t in enumerate(terms):
        vp[:, 1 + i] = -t[:, None]
    q = torch.zeros(B, hq * d, dtype=torch.bfloat16, device="cuda")
    q[:, ::d] = 1.0
    kp, vp = (t.bfloat16().cuda() for t in (kp, vp))
    got = ops.attention_decode_paged(q, kp, vp, torch.arange(B, dtype=I32, device="cuda")[:, None].contiguous(), torch.full((B,), 4, dtype=I32, device="cuda"), hq, hk, d, scale=1.0)
    got, w = got.double().cpu(), w[:, None]
    bound = (1.5 * 2.0 ** -22 * w + 4 * 2.0 ** -23 + left.abs()[:, None]) / (3 + w) * (1 + 2.0 ** -8)
    assert (got.abs() <= bound).all(), float((got.abs() / bound).max())


def test_attention_repeats_bit_for_bit_and_on_another_stream():
    import plz_ops as ops
    a = _case(1, RAGGED * 3, 32, 8, 128, 16)
    first = ops.attention_decode_paged(*a, 32, 8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = ops.attention_decode_paged(*a, 32, 8)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first, second) and torch.equal(first, ops.attention_decode_paged(*a, 32, 8))


def test_captured_attention_follows_the_lengths():
    """Two captured calls with a workspace each, replayed in turns after lengths and tables changed."""
    import plz_ops as ops
    a, b = _case(1, [500, 20, 90, 1], 8, 2, 128, 16), _case(2, [64, 900], 8, 2, 64, 8)
    calls = [lambda: ops.attention_decode_paged(*a, 8, 2), lambda: ops.attention_decode_paged(*b, 8, 2, 64)]
    for f in calls:
        f()
    graphs, outs = [], []
    for f in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    for change in range(3):
        for i in (0, 1, 1, 0):
            graphs[i].replay()
        _close(outs[0], *ref.attention(*a, 8, 2, 128))
        _close(outs[1], *ref.attention(*b, 8, 2, 64))
        a[4].copy_(_dev([[16, 20, 0, 1], [333, 5, 90, 0]][change % 2]))
        b[4].copy_(_dev([1, 17 + change]))


def test_no_requests():
    import plz_ops as ops
    q, kp, vp, table, L = _case(1, [5], 8, 2, 128, 16)
    assert ops.attention_decode_paged(q[:0], kp, vp, table[:0], L[:0], 8, 2).shape == (0, 1024)
    L.zero_()
    assert (ops.attention_decode_paged(q, kp[:0], vp[:0], table[:, :0], L, 8, 2) == 0).all()


@pytest.mark.parametrize("lengths", [[16] * 700, [9000, 5, 9000], [2049], [40] * 33], ids=["by a warp", "across CTAs", "one request", "small batch"])
@pytest.mark.parametrize("page", [0, 2 ** 31 - 1, -1])
def test_requests_without_any_page_in_the_pool(page, lengths):
    """No weight at all: NaN in their rows wherever they are finished, the others as they are."""
    import plz_ops as ops
    q, kp, vp, table, L = _case(len(lengths), lengths, 8, 2, 128, 16)
    want, err = ref.attention(q, kp, vp, table, L, 8, 2, 128)
    gone = torch.arange(len(lengths)) % 2 == 0
    table[gone.cuda()] = page if page else kp.shape[0]
    bad = torch.zeros(1, dtype=I32, device="cuda")
    got = ops.attention_decode_paged(q, kp, vp, table, L, 8, 2, bad=bad)
    check_status()
    assert got[gone.cuda()].isnan().all() and bad.item() == 1
    if not gone.all():
        _close(got.cpu()[~gone], want.cpu()[~gone], err.cpu()[~gone])


def test_lengths_next_to_the_largest_number():
    """A table with room for 2^31 tokens, all of them one page: lengths up to 2^31 - 64 are served, longer ones cut to that. Equal weights over the page's values, sums of them whole."""
    import plz_ops as ops
    page, most = 1 << 16, 2 ** 31 - 64
    kp = torch.zeros(1, page, 64, dtype=torch.bfloat16, device="cuda")
    vp = torch.ones_like(kp)
    vp[:, :, 1] = -2.0
    table = torch.zeros(1, 1 << 15, dtype=I32, device="cuda")
    q = torch.ones(1, 128, dtype=torch.bfloat16, device="cuda")
    bad = torch.zeros(1, dtype=I32, device="cuda")
    for n, cut in ((most - 1, 0), (most, 0), (most + 1, 1), (2 ** 31 - 1, 1)):
        got = ops.attention_decode_paged(q, kp, vp, table, _dev([n]), 2, 1, 64, bad=bad).view(2, 64)
        assert bad.item() == cut and (got[:, 0] == 1).all() and (got[:, 1] == -2).all() and (got[:, 2:] == 1).all(), n
        bad.zero_()


def test_pool_past_four_gigabytes():
    """Offsets that no 32-bit count of elements or bytes holds: the request's pages lie at both ends of a pool of 6 GB per tensor."""
    import plz_ops as ops
    page, W = 64, 256
    n_pages = 6 * 2 ** 30 // (page * W * 2)
    kp, vp = (torch.zeros(n_pages, page, W, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.tensor([[n_pages - 1, 0, n_pages // 2 + 3, n_pages - 2]], dtype=I32, device="cuda")
    n = 230
    k, v = (torch.randn(n, W, generator=g, device="cuda").bfloat16() for _ in range(2))
    plan = ops.plan_pages(_dev([0]), _dev([n]), torch.full((1, 4), -1, dtype=I32, device="cuda"), ids.flip(1).view(-1).contiguous(), _dev([4]), page, n)
    pos = torch.arange(n, device="cuda")
    slots = (ids[0, pos // page].long() * page + pos % page).to(I32)
    del plan
    ops.write_pages(k, v, slots, kp, vp)
    q = torch.randn(1, 8 * 128, generator=g, device="cuda").bfloat16()
    got = ops.attention_decode_paged(q, kp, vp, ids, _dev([n]), 8, 2)
    small = [t[ids[0].long()].contiguous() for t in (kp, vp)]
    _close(got, *ref.attention(q, *small, _dev([[0, 1, 2, 3]]), _dev([n]), 8, 2, 128))


# ---- the calls from Python -----------------------------------------------------------------------------------------------------
class _Declines:
    """In place of the native calls: declines everything, so that the general path runs."""
    def __getattr__(self, name):
        return lambda *a: None


def test_general_path_and_native_calls_agree(monkeypatch):
    import plz_native as P
    import plz_ops as ops
    import seq_ops as S

    def everything():
        cached, new, table, free, n_free = _requests(5, 30, 16, 100, 9, spare=60, ended=0.1)
        tab, F = _dev(table), _dev(free)
        p = ops.plan_pages(_dev(cached), _dev(new), tab, F, _dev([n_free]), 16, 200)
        q, kp, vp, t2, L = _case(4, RAGGED, 8, 2, 128, 16, fill=0.0)
        k = torch.arange(13 * 256, device="cuda").view(13, 256).bfloat16()
        slots = torch.arange(13, device="cuda", dtype=I32) * 3 - 1
        ops.write_pages(k, k * 2, slots, kp, vp)
        out = torch.zeros(13, 1104, dtype=torch.bfloat16, device="cuda")[:, 8:1032]
        bad = torch.zeros(1, dtype=I32, device="cuda")
        o1, o2 = ops.attention_decode_paged(q, kp, vp, t2, L, 8, 2), ops.attention_decode_paged(q, kp, vp, t2, L, 8, 2, 128, 0.5, out, bad)
        g = torch.Generator(device="cuda").manual_seed(1)
        x = torch.randn(3, 500, generator=g, device="cuda")
        tok = torch.randint(0, 500, (3, 40), generator=g, device="cuda")
        one = torch.full((3,), 1.5, device="cuda")
        kw = dict(tokens=tok, lengths=_dev([40, 3, 0]), prompt_lengths=_dev([4, 0, 1]), repetition=one, presence=0.5, frequency=0, bias_ids=tok[:, :7].contiguous(), bias=torch.randn(3, 7, generator=g, device="cuda"),
                  mask=torch.randint(-2 ** 31, 2 ** 31, (1, 16), generator=g, device="cuda").int())
        y1, y2 = S.adjust_logits(x, **kw), S.adjust_logits(x.bfloat16(), presence=0.25, tokens=tok, lengths=_dev([40, 3, 0]))
        y3 = S.adjust_logits(x, out=torch.empty_like(x))
        return [p.lengths, p.n_free, p.starts, p.slots, p.positions, p.status, tab, F, kp, vp, o1, o2, out.clone(), bad, y1, y2, y3]
    native = everything()
    calls = P.calls()
    for name in ("plan_pages", "write_pages", "attention_decode_paged", "adjust_logits"):
        assert getattr(calls, name)() is None
    monkeypatch.setattr(P, "calls", lambda: _Declines())
    general = everything()
    assert all(torch.equal(a, b) for a, b in zip(native, general))
    # a tensor on another device than the current one is refused ahead of any launch
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    with pytest.raises(P.PlzError, match="current device"):
        everything()


def test_results_of_a_plan_have_storages_of_their_own():
    """Growing one of them leaves the others as they are, and saving one saves no more than it."""
    import plz_ops as ops
    p = ops.plan_pages(_dev([3, 0]), _dev([2, 5]), _dev([[4, -1], [-1, -1]]), _dev([0, 1, 2, 3, -1]), _dev([4]), 4, 8)
    parts = (p.lengths, p.n_free, p.starts, p.slots, p.positions, p.status)
    assert len({t.untyped_storage().data_ptr() for t in parts}) == 6
    assert all(t.storage_offset() == 0 and t.untyped_storage().nbytes() == 4 * t.numel() for t in parts)
    positions = p.positions.clone()
    p.slots.resize_(16).fill_(99)
    assert torch.equal(p.positions, positions)


def test_results_that_are_written_past_are_refused():
    import plz_native as P
    import plz_ops as ops
    q, kp, vp, table, L = _case(1, [5], 8, 2, 128, 16)
    with pytest.raises(P.PlzError):
        ops.attention_decode_paged(q, kp, vp, table, L, 8, 2, out=q)
    new = _dev([1])
    with pytest.raises(P.PlzError):
        ops.plan_pages(L, new, table, _dev([0]), _dev([1]), 16, 1, lengths_out=new)
    with pytest.raises(P.PlzError):          # rows that are no whole 16-byte units
        ops.write_pages(kp[0, :, :100], vp[0, :, :100], _dev([-1] * 16), kp[:, :, :100], vp[:, :, :100])
