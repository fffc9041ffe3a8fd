"""What the operators of a batch of requests refuse, on the host ahead of any launch, and the plain statements that their tests compare with."""
import ctypes as C

import pytest
import torch

import paged_cases as ref

OK, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE, NULL, LARGE = 0, 1, 2, 3, 5, 7, 8
PTR = 0x10000


def _call(fn, cls, base, lead=(), tail=(None,)):
    def call(**kw):
        return fn(*lead, C.byref(cls(**{**base, **kw})), *tail)
    return call


def test_page_plan_refusals(built_lib):
    import plz_native as P
    base = {n: PTR + 0x1000 * i for i, (n, t) in enumerate(P.PagePlan._fields_) if t is C.c_void_p}
    call = _call(P.lib().plz_page_plan, P.PagePlan, {**base, "ldt": 8, "B": 4, "width": 8, "page_size": 16, "n_pages": 100, "max_rows": 4, "row_pitch": 0})
    for name in base:
        assert call(**{name: None}) == NULL, name
    assert P.lib().plz_page_plan(None, None) == NULL
    for kw in ({"B": -1}, {"width": -1}, {"page_size": 0}, {"n_pages": -1}, {"max_rows": -1}, {"row_pitch": -1}, {"ldt": 7}):
        assert call(**kw) == SHAPE, kw
    for kw in ({"B": 16385}, {"width": 1 << 28, "ldt": 1 << 28}, {"n_pages": 1 << 27}, {"max_rows": (1 << 30) + 1}):
        assert call(**kw) == LARGE, kw
    assert b"16384" in P.lib().plz_last_error()
    assert call(lengths=base["new_tokens"]) == UNSUPPORTED


def test_page_plan_refuses_a_status_over_its_inputs(built_lib):
    import plz_native as P
    import plz_ops as ops
    base = {n: PTR + 0x1000 * i for i, (n, t) in enumerate(P.PagePlan._fields_) if t is C.c_void_p}
    call = _call(P.lib().plz_page_plan, P.PagePlan, {**base, "ldt": 8, "B": 4, "width": 8, "page_size": 16, "n_pages": 100, "max_rows": 4, "row_pitch": 0})
    assert [call(status=base[name]) for name in ("new_tokens", "cached", "lengths")] == [UNSUPPORTED] * 3
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for wrong in (i32(2), i32(3).long()):
        with pytest.raises(AssertionError):
            ops.plan_pages(i32(3), i32(3), i32(3, 4), i32(9), i32(1), 16, 3, status_out=wrong)


def test_page_plan_refuses_a_negative_limit(built_lib):
    import plz_native as P
    base = {n: PTR + 0x1000 * i for i, (n, t) in enumerate(P.PagePlan._fields_) if t is C.c_void_p}
    assert _call(P.lib().plz_page_plan, P.PagePlan, {**base, "ldt": 8, "B": 4, "width": 8, "page_size": 16, "n_pages": 100, "max_rows": 4, "row_pitch": 0})(max_tokens=-1) == SHAPE


def test_page_write_refusals(built_lib):
    import plz_native as P
    base = dict(k=PTR, v=PTR, ldk=64, ldv=64, k_pages=PTR, v_pages=PTR, page_stride=1024, tok_stride=64, slots=PTR, rows=3, row_bytes=64, page_size=16, n_pages=5)
    call = _call(P.lib().plz_page_write, P.PageWrite, base)
    assert call(rows=0) == OK and call(n_pages=0) == OK and call(rows=0, k=None) == OK
    for name in ("k", "v", "k_pages", "v_pages", "slots"):
        assert call(**{name: None}) == NULL, name
    for kw in ({"rows": -1}, {"row_bytes": 0}, {"page_size": 0}, {"n_pages": -1}, {"ldk": -64}, {"tok_stride": 48}, {"page_stride": 48}):
        assert call(**kw) == SHAPE, kw
    for kw in ({"k": PTR + 8}, {"v_pages": PTR + 2}, {"ldv": 72}, {"row_bytes": 40}, {"tok_stride": 72}, {"page_stride": 1028}):
        assert call(**kw) == ALIGN, kw
    assert call(n_pages=1 << 28) == LARGE and call(rows=(1 << 30) + 1) == LARGE


def test_paged_attention_refusals(built_lib):
    import plz_native as P
    lib = P.lib()
    base = dict(q=PTR, ldq=1024, k_pages=PTR, v_pages=PTR, page_stride=4096, tok_stride=256, table=PTR, ldt=8, lengths=PTR, out=2 * PTR, ldo=1024, bad=None, B=3, width=8, page_size=16, n_pages=5,
                Hq=8, Hkv=2, head_dim=128, scale=1.0)
    need = lib.plz_attn_decode_paged_ws_bytes(8, 2, 128)
    assert need > 0 and lib.plz_attn_decode_paged_ws_bytes(0, 2, 128) == 0 and lib.plz_attn_decode_paged_ws_bytes(32, 2, 128) > need
    call = _call(lib.plz_attn_decode_paged, P.AttnDecodePaged, base, tail=(PTR, need, None))
    assert call(B=0) == OK
    for name in ("q", "k_pages", "v_pages", "table", "lengths", "out"):
        assert call(**{name: None}) == NULL, name
    for kw in ({"B": -1}, {"Hq": 7}, {"Hkv": 0}, {"head_dim": 96}, {"head_dim": 0}, {"page_size": 0}, {"width": -1}, {"n_pages": -1}, {"ldq": 1016}, {"ldo": 0}, {"ldt": 7}, {"tok_stride": 248},
               {"page_stride": 128}):
        assert call(**kw) == SHAPE, kw
    for kw in ({"q": PTR + 2}, {"out": 2 * PTR + 8}, {"k_pages": PTR + 4}, {"ldq": 1028}, {"tok_stride": 260}, {"page_stride": 4100}):
        assert call(**kw) == ALIGN, kw
    assert call(page_stride=1 << 36) == LARGE and call(page_stride=1 << 33, n_pages=40) == LARGE
    assert call(out=PTR) == UNSUPPORTED
    assert _call(lib.plz_attn_decode_paged, P.AttnDecodePaged, base, tail=(PTR + 8, need, None))() == ALIGN
    for ws in ((PTR, need - 1, None), (None, need, None)):
        assert _call(lib.plz_attn_decode_paged, P.AttnDecodePaged, base, tail=ws)() == WORKSPACE


def test_adjust_logits_refusals(built_lib):
    import plz_native as P
    base = dict(logits=PTR, ld=100, out=PTR, ldo=100, tokens=PTR, ldk=9, lengths=PTR, prompt_lengths=None, repetition=None, presence=None, frequency=None, bias_ids=PTR, bias=PTR, ldb=3, mask=PTR, ldm=4,
                repetition_all=1.0, presence_all=0.0, frequency_all=0.0, rows=2, V=100, max_tokens=9, n_bias=3)
    call = _call(P.lib().plz_adjust_logits, P.AdjustLogits, base, lead=(1,))
    assert call(rows=0) == OK
    assert _call(P.lib().plz_adjust_logits, P.AdjustLogits, base, lead=(2,))() == UNSUPPORTED
    for name in ("logits", "out", "tokens", "bias_ids", "bias"):
        assert call(**{name: None}) == NULL, name
    for kw in ({"rows": -1}, {"V": 0}, {"ld": 99}, {"ldo": 99}, {"ldk": 8}, {"ldb": 2}, {"ldm": 3}, {"max_tokens": -1}, {"n_bias": -1}, {"ldk": -1}):
        assert call(**kw) == SHAPE, kw
    for kw in ({"rows": 65536}, {"n_bias": 4097, "ldb": 5000}, {"max_tokens": 1 << 30, "ldk": 1 << 30}):
        assert call(**kw) == LARGE, kw
    assert call(logits=PTR + 2) == ALIGN


def test_adjust_logits_in_place_with_two_pitches(built_lib):
    """Over the logits themselves, but with rows that lie elsewhere: a row's results would go over another row's logits."""
    import plz_native as P
    base = dict(logits=PTR, ld=100, out=PTR, ldo=104, tokens=None, ldk=0, lengths=None, prompt_lengths=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None, ldb=0, mask=None,
                ldm=0, repetition_all=1.0, presence_all=0.0, frequency_all=0.0, rows=2, V=100, max_tokens=0, n_bias=0)
    call = _call(P.lib().plz_adjust_logits, P.AdjustLogits, base, lead=(1,))
    assert call(rows=0) == OK and call() == UNSUPPORTED and call(ld=104, ldo=100) == UNSUPPORTED


def test_binding_refusals(built_lib):
    """Types and shapes that the binding passes as bare pointers, and tensors that are not on a GPU."""
    import plz_native as P
    import plz_ops as ops
    import seq_ops as S
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    plan = dict(lengths=i32(3), new_tokens=i32(3), table=i32(3, 4), free_pages=i32(9), n_free=i32(1), page_size=16, max_rows=3)
    write = dict(k=bf(3, 64), v=bf(3, 64), slots=i32(3), k_pages=bf(5, 16, 64), v_pages=bf(5, 16, 64))
    attn = dict(q=bf(3, 512), k_pages=bf(5, 16, 128), v_pages=bf(5, 16, 128), table=i32(3, 4), lengths=i32(3), n_heads=4, n_kv_heads=1)
    logits = dict(logits=torch.zeros(3, 50), tokens=torch.zeros(3, 7, dtype=torch.int64), lengths=i32(3), bias_ids=torch.zeros(3, 2, dtype=torch.int64), bias=torch.zeros(3, 2), mask=i32(3, 2))
    for f, good, wrong in (
            (ops.plan_pages, plan, ({"lengths": i32(3).long()}, {"new_tokens": i32(4)}, {"table": i32(2, 4)}, {"table": i32(4, 3).t()}, {"n_free": i32(2)}, {"free_pages": i32(9, 1)}, {"lengths_out": i32(2)})),
            (ops.write_pages, write, ({"k": bf(3, 64).float()}, {"v": bf(2, 64)}, {"slots": i32(3).long()}, {"k_pages": bf(5, 16, 32)}, {"v_pages": bf(5, 8, 64)}, {"k": bf(64, 3).t(), "v": bf(64, 3).t()})),
            (ops.attention_decode_paged, attn, ({"lengths": i32(2)}, {"table": i32(3, 4).long()}, {"bad": i32(2)}, {"out": bf(2, 512)})),
            (S.adjust_logits, logits, ({"logits": torch.zeros(3, 50).double()}, {"tokens": i32(3, 7)}, {"lengths": None}, {"lengths": i32(3).long()}, {"bias": None}, {"bias": torch.zeros(3, 3)},
                                       {"bias": torch.zeros(3, 4)[:, :2]}, {"mask": i32(3, 3)}, {"mask": i32(2, 2)}, {"repetition": torch.zeros(3).double()}, {"presence": torch.zeros(1)},
                                       {"prompt_lengths": i32(4)}, {"out": torch.zeros(3, 51)}))):
        with pytest.raises(P.PlzError):          # right in everything, but in host memory
            f(**good)
        for kw in wrong:
            with pytest.raises((AssertionError, KeyError)):
                f(**{**good, **kw})


def test_tokens_in_host_memory_are_refused_ahead_of_the_library(built_lib):
    import plz_native as P
    import plz_ops as ops
    with pytest.raises(P.PlzError, match="CUDA tensors only"):
        ops.embed_gather(torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64))


def test_settings_that_make_no_number_are_refused_with_the_request(built_lib):
    from types import SimpleNamespace
    from engine import Engine, SamplingParams
    eng = Engine(SimpleNamespace(vocab=100), 64)
    nan, inf = float("nan"), float("inf")
    for kw in ({"repetition": nan}, {"repetition": inf}, {"repetition": 1e39}, {"repetition": 1e-46}, {"repetition": -1.0}, {"presence": nan}, {"frequency": nan}, {"presence": inf, "frequency": -inf},
               {"presence": 1e39, "frequency": -1e39}, {"bias": ((3, nan),)}, {"bias": ((3, inf), (3, -inf))}, {"bias": ((3, inf),), "presence": inf}):
        with pytest.raises(ValueError):
            eng.submit([1], SamplingParams(**kw))
    assert not eng.waiting
    for kw in ({"repetition": 1e38}, {"repetition": 1e-45}, {"presence": inf}, {"frequency": -3.0}, {"bias": ((3, -inf), (4, inf), (3, 1.0))}, {"bias": ((3, -inf),), "presence": inf}):
        eng.submit([1], SamplingParams(**kw))


def test_the_plain_plan():
    """By hand: two requests that share five free pages with one that ends, and a third that comes too late."""
    table, free = [[4, -1, -1], [7, 8, -1], [-1, -1, -1], [9, -1, -1]], [0, 1, 2, 3, 5, -1, -1, -1, -1, -1]
    lengths, left, starts, slots, positions, status = ref.plan([3, 5, 0, 2], [6, -1, 9, 1], table, free, 5, 4, 20)
    assert starts == [0, 6, 6, 15, 16] and lengths == [9, 0, 9, 3] and status == [0, 0, 0, 0]
    assert table[0] == [4, 5, 3] and table[2] == [2, 1, 0] and left == 2 and free[:2] == [7, 8]
    assert slots[:6] == [19, 20, 21, 22, 23, 12] and slots[6:15] == [8, 9, 10, 11, 4, 5, 6, 7, 0] and slots[15] == 38 and slots[16:] == [-1] * 4
    assert positions[:6] == [3, 4, 5, 6, 7, 8] and positions[15:] == [2, -1, -1, -1, -1]
    assert ref.plan([0, 0, 0], [9, 5, 0], [[-1] * 3 for _ in range(3)], [0, 1, 2, 3], 4, 4, 20)[5] == [0, 1, 0]
