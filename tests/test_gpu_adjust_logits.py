"""Penalties, biases and grammar masks on logits, against the formula in 64 bits."""
import pytest
import torch

import paged_cases as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


def _inputs(seed, rows, V, n_tok, n_bias, mask, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ri = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda")
    x = (4 * torch.randn(rows, V, generator=g, device="cuda")).to(dtype)
    kw = {}
    if n_tok:
        kw["tokens"] = (torch.rand(rows, n_tok, generator=g, device="cuda") ** 3 * V).long().clamp(max=V - 1)
        kw["tokens"][:, n_tok // 2] = V + 5            # nobody's
        kw["tokens"][:, n_tok // 3] = -1
        kw["lengths"] = ri(0, n_tok + 1, rows).int()
        kw["lengths"][0] = n_tok
        kw["prompt_lengths"] = ri(0, n_tok + 1, rows).int()
        kw.update(repetition=0.5 + torch.rand(rows, generator=g, device="cuda"), presence=torch.randn(rows, generator=g, device="cuda"), frequency=torch.randn(rows, generator=g, device="cuda"))
    if n_bias:
        kw["bias_ids"] = ri(-2, V + 2, rows, n_bias)
        kw["bias_ids"][:, -1] = kw["bias_ids"][:, 0]   # one token twice
        kw["bias"] = torch.randn(rows, n_bias, generator=g, device="cuda")
    if mask:
        kw["mask"] = ri(-2 ** 31, 2 ** 31, rows, (V + 31) // 32).int()
        kw["mask"][-1] = 0 if rows > 1 else kw["mask"][-1]
    return x, kw


def _check(got, x, kw):
    names = {"prompt_lengths": "prompt", "repetition": "rep", "presence": "pres", "frequency": "freq"}
    want, size = ref.adjust(x, **{names.get(k, k): v for k, v in kw.items()})
    got = got.double().cpu()
    off = torch.isinf(want)
    assert torch.equal(got[off], want[off])
    # eight operations ahead of the last rounding, each off by 2^-24 of the sizes added up
    err = 8 * 2.0 ** -24 * size + (2.0 ** -8 * want.abs() if x.dtype == torch.bfloat16 else 0)
    assert ((got - want).abs() <= err)[~off].all(), float(((got - want).abs() - err)[~off].max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", [(1, 1), (1, 31), (3, 33), (2, 1001), (5, 32768), (2, 50257), (3, 151936), (70, 515)])
@pytest.mark.parametrize("n_tok,n_bias,mask", [(0, 0, True), (300, 0, False), (0, 40, False), (777, 33, True)])
def test_adjust(rows, V, n_tok, n_bias, mask, dtype):
    import seq_ops as S
    x, kw = _inputs(rows * V + n_tok, rows, V, n_tok, n_bias, mask, dtype)
    keep = x.clone()
    got = S.adjust_logits(x, **kw)
    assert torch.equal(x, keep) and got.dtype == dtype
    _check(got, x, kw)
    assert torch.equal(got, S.adjust_logits(x, **kw))
    S.adjust_logits(x, out=x, **kw)
    assert torch.equal(x, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_tok", [8191, 8192, 8193, 20000])
def test_long_histories(n_tok, dtype):
    """Both sides of the line between the two widths of counts, one row that says a single token all the time."""
    import seq_ops as S
    x, kw = _inputs(n_tok, 3, 50257, n_tok, 20, True, dtype)
    kw["tokens"][1] = 50256
    kw["lengths"][1], kw["prompt_lengths"][1] = n_tok, 3
    kw["frequency"][1] = 2.0 ** -12
    _check(S.adjust_logits(x, **kw), x, kw)


@pytest.mark.parametrize("rows,V,n_bias", [(1, 1000003, 50), (300, 40970, 5), (150, 82000, 0), (2, 163841, 4096)])
def test_vocabularies_of_many_segments(rows, V, n_bias):
    import seq_ops as S
    x, kw = _inputs(rows, rows, V, 100, n_bias, True, torch.bfloat16)
    kw["tokens"][:, :4] = torch.tensor([0, V - 1, V // 2, 7], device="cuda")
    _check(S.adjust_logits(x, **kw), x, kw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Pitched and shifted logits and results (whole rows off the 16-byte grid, both alike and not), pitched tokens and biases, one mask for all rows, numbers for all rows."""
    import seq_ops as S
    rows, V = 3, 9001
    x, kw = _inputs(1, rows, V, 100, 10, True, dtype)
    for shift_in, shift_out in ((0, 0), (1, 1), (3, 1), (5, 0)):
        a = torch.zeros(rows, V + 13, dtype=dtype, device="cuda")[:, shift_in:shift_in + V]
        a.copy_(x)
        room = torch.full((rows, V + 13), 3.0, dtype=dtype, device="cuda")
        wide = {k: torch.nn.functional.pad(kw[k], (2, 5))[:, 2:-5] for k in ("tokens", "bias_ids", "bias", "mask")}
        S.adjust_logits(a, out=room[:, shift_out:shift_out + V], **{**kw, **wide})
        _check(room[:, shift_out:shift_out + V], x, kw)
        assert (room[:, :shift_out] == 3).all() and (room[:, shift_out + V:] == 3).all()
    shared = {**kw, "mask": kw["mask"][:1], "repetition": 1.3, "presence": 0.25, "frequency": -0.5}
    _check(S.adjust_logits(x, **shared), x, shared)
    del shared["prompt_lengths"]
    _check(S.adjust_logits(x, **shared), x, shared)
    every = {**kw, "tokens": kw["tokens"][:1].expand(rows, -1), "bias_ids": kw["bias_ids"][:1].expand(rows, -1), "bias": kw["bias"][:1].expand(rows, -1)}
    _check(S.adjust_logits(x, **every), x, every)


def test_lengths_past_the_tokens_and_below_none():
    import seq_ops as S
    x, kw = _inputs(2, 4, 500, 20, 0, False, torch.float32)
    kw["lengths"] = torch.tensor([-3, 21, 2 ** 31 - 1, 0], dtype=torch.int32, device="cuda")
    kw["prompt_lengths"] = torch.tensor([-3, -1, 5, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    _check(S.adjust_logits(x, **kw), x, kw)


def test_logits_that_are_no_numbers_stay_so():
    import seq_ops as S
    x = torch.tensor([[float("inf"), float("-inf"), float("nan"), 1.0, -0.0]], device="cuda")
    tok = torch.arange(5, device="cuda").view(1, 5)
    got = S.adjust_logits(x, tokens=tok, lengths=torch.tensor([5], dtype=torch.int32, device="cuda"), repetition=2.0, presence=1.0)[0].tolist()
    assert got[0] == float("inf") and got[1] == float("-inf") and got[2] != got[2] and got[3] == -0.5 and got[4] == -1.0


def test_repetition_is_one_rounded_operation():
    """x / r and x * r as fp32 makes them, to the last bit, for factors whose inverse has no fp32 value too."""
    import seq_ops as S
    factors = [1.1, 1.3, 1.7, 3.0, 0.7, 1e-39, 2.0 ** -149, 3e38, 1e30]
    V = 4099
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(len(factors), V, generator=g, device="cuda") * torch.tensor([1, 1, 1, 1, 1, 1e-3, 1e-10, 1e30, 1e30], device="cuda")[:, None]
    r = torch.tensor(factors, device="cuda")
    tok = torch.arange(V, device="cuda").expand(len(factors), -1)
    got = S.adjust_logits(x, tokens=tok, lengths=torch.full((len(factors),), V, dtype=torch.int32, device="cuda"), repetition=r)
    x, r = x.cpu(), r.cpu()[:, None]
    want = torch.where(x > 0, x / r, x * r)
    assert torch.isfinite(want[5]).all() and torch.equal(got.cpu(), want)


def test_a_token_said_very_often_and_every_token_biased():
    import seq_ops as S
    V, n = 700, 100000
    x = torch.zeros(2, V, device="cuda")
    tok = torch.zeros(2, n, dtype=torch.int64, device="cuda")
    tok[1] = 699
    ids = torch.arange(V, device="cuda").repeat(2, 5)
    b = torch.randn(2, 5 * V, device="cuda")
    kw = dict(tokens=tok, lengths=torch.tensor([n, n - 1], dtype=torch.int32, device="cuda"), frequency=0.01, bias_ids=ids, bias=b)
    got = S.adjust_logits(x, **kw)
    _check(got, x, kw)


def test_captured_and_no_rows():
    import seq_ops as S
    x, kw = _inputs(3, 4, 3000, 64, 8, True, torch.float32)
    S.adjust_logits(x, **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = S.adjust_logits(x, **kw)
    kw["lengths"].fill_(64)
    kw["tokens"].add_(1)
    x.mul_(-1)
    g.replay()
    _check(out, x, kw)
    assert S.adjust_logits(x[:0]).shape == (0, 3000)


def test_masked_tokens_are_never_picked():
    import seq_ops as S
    rows, V = 4, 2000
    x = torch.randn(rows, V, device="cuda")
    allowed = [3, 1999, 777, 64]
    mask = torch.zeros(rows, (V + 31) // 32, dtype=torch.int64)
    for r, t in enumerate(allowed):
        mask[r, t // 32] = 1 << (t % 32)
    mask = torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).int().cuda()
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    for temperature, top_k in ((0.0, 0), (1.0, 0), (0.7, 5)):
        assert S.sample(S.adjust_logits(x, mask=mask), pos, temperature, top_k, 3).tolist() == allowed
