"""The paged operators as a served model uses them: a batch of requests of different lengths decoded together, against each request alone over a cache of its own, and the
settings of a request in the engine."""
import pytest
import torch

from helpers import assert_close, check_status

pytestmark = pytest.mark.gpu
CFG = dict(hidden=512, n_heads=8, n_kv_heads=2, intermediate=1024, n_layers=2, vocab=1000)


def _model(seed=0, **kw):
    import decode_model as D
    return D.PalettizedQwen.random(D.ModelConfig(**{**CFG, **kw}), torch.device("cuda", 0), seed=seed, max_positions=512)


@pytest.mark.parametrize("page_size", [16, 24])
@pytest.mark.parametrize("B", [5, 70])
def test_requests_of_different_lengths(B, page_size):
    """Prompts filled in, tokens decoded with some requests idle, one ended and its row used again: logits equal those of every request alone."""
    m = _model()
    g = torch.Generator().manual_seed(B)
    prompts = [torch.randint(0, 1000, (128 * (b % 3) + (b * 7) % 5,), generator=g) for b in range(B)]
    cache = m.new_paged_cache(B, n_pages=B * -(-300 // page_size), page_size=page_size, max_tokens=300)
    alone = [m.new_cache(1, 300) for _ in range(B)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for n in (128, 256):
        rows = [b for b in range(B) if len(prompts[b]) // 128 * 128 == n]
        if rows:
            kv = m.new_cache(len(rows), n)
            m.prefill(torch.stack([prompts[b][:n] for b in rows]).cuda(), kv, want_logits=False)
            assert not cache.fill(kv, rows).status.any()
    for b in range(B):
        n = len(prompts[b]) // 128 * 128
        if n:
            m.prefill(prompts[b][None, :n].cuda(), alone[b], want_logits=False)

    def step(tokens):
        """tokens: per request an id, None (idle) or -1 (ended)."""
        ids = torch.tensor([t if t is not None and t >= 0 else 0 for t in tokens], device="cuda")
        got = m.decode_paged(ids, cache, i32([0 if t is None else 1 if t >= 0 else -1 for t in tokens]))
        live = [b for b in range(B) if tokens[b] is not None and tokens[b] >= 0]
        for b in range(B):
            if tokens[b] == -1:
                alone[b].reset()
        want = torch.cat([m.decode_step(torch.tensor([tokens[b]], device="cuda"), alone[b]) for b in live])
        assert_close(got[live], want, "logits", rel=3e-2, cos=0.999)
        assert cache.lengths.tolist() == [c.length for c in alone]
    tails = [prompts[b][len(prompts[b]) // 128 * 128:].tolist() for b in range(B)]
    for t in range(4):
        step([tails[b][t] if t < len(tails[b]) else None if b else 5 for b in range(B)])
    for t in range(6):
        tok = torch.randint(0, 1000, (B,), generator=g).tolist()
        step([None if (b + t) % 4 == 0 and b else -1 if t == 2 and b == B - 1 else tok[b] for b in range(B)])
    check_status()
    held = -(-cache.lengths // page_size)
    used = torch.cat([cache.table[b, :n] for b, n in enumerate(held.tolist())] + [cache.free_pages[:cache.n_free.item()]])
    assert sorted(used.tolist()) == list(range(cache.free_pages.shape[0]))      # every page belongs to one request or is free


def test_a_captured_step_replays():
    m = _model(1)
    B = 4
    a, b = (m.new_paged_cache(B, n_pages=60, page_size=8, max_tokens=100) for _ in range(2))
    ids, new = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    m.decode_paged(ids, a, new)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.decode_paged(ids, a, new)
    g = torch.Generator().manual_seed(3)
    for t in range(20):
        ids.copy_(torch.randint(0, 1000, (B,), generator=g))
        new.copy_(torch.tensor([1, t % 2, 1 if t != 9 else -1, int(t > 5)], dtype=torch.int32))
        graph.replay()
        want = m.decode_paged(ids, b, new)
        live = new > 0
        # the products of up to 16 rows add partial sums with atomics: bits may differ between runs, as in the model's other steps
        assert_close(out[live], want[live], "logits", rel=3e-2, cos=0.999)
        assert torch.equal(a.lengths, b.lengths) and torch.equal(a.table, b.table)


def test_more_tokens_than_the_model_has_positions_are_refused():
    m = _model(1)
    c = m.new_paged_cache(2, 10, 16, 528)
    with pytest.raises(ValueError):
        m.decode_paged(torch.zeros(2, dtype=torch.int64, device="cuda"), c, torch.ones(2, dtype=torch.int32, device="cuda"))
    c = m.new_paged_cache(2, 10, 16, 64)
    for ids, new in ((3, 2), (2, 1)):
        with pytest.raises(ValueError):
            m.decode_paged(torch.zeros(ids, dtype=torch.int64, device="cuda"), c, torch.ones(new, dtype=torch.int32, device="cuda"))
    for rows in ([0], [0, 0], [1, 0], [0, 2]):
        with pytest.raises(ValueError):
            c.fill(m.new_cache(2, 128), rows)


@pytest.mark.parametrize("captured", [False, True])
def test_a_step_without_a_page_for_a_request_is_told(captured):
    """Three requests, pages for two: who got none is told by the cache's status, keeps its length, and goes on as if nothing had been once another one has ended."""
    m = _model(4)
    B, page = 3, 4
    cache = m.new_paged_cache(B, n_pages=4, page_size=page, max_tokens=64)
    alone = [m.new_cache(1, 64) for _ in range(B)]
    ids, new = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    status = cache.status
    step = lambda: m.decode_paged(ids, cache, new)
    if captured:
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        step = lambda: (graph.replay(), out)[1]
    g = torch.Generator().manual_seed(6)
    tokens = torch.randint(0, 1000, (B, 20), generator=g).tolist()
    at, seen = [0] * B, []
    for t in range(10):
        bring = [-1 if t == 7 else int(t < 7), 1, 1]
        ids.copy_(torch.tensor([tokens[b][at[b]] for b in range(B)]))
        new.copy_(torch.tensor(bring, dtype=torch.int32))
        got = step()
        told = status.tolist()
        seen.append(told)
        for b in range(B):
            if bring[b] < 0:
                alone[b].reset()
                at[b] = 0
            elif bring[b] and told[b] == 0:
                assert_close(got[b:b + 1], m.decode_step(torch.tensor([tokens[b][at[b]]], device="cuda"), alone[b]), "logits", rel=3e-2, cos=0.999)
                at[b] += 1
        assert cache.lengths.tolist() == at and cache.status is status
    # four pages: one each for the first four tokens, one for request 0's fifth; the others wait until it has ended and gave two back
    assert seen == [[0, 0, 0]] * 4 + [[0, 1, 1]] * 4 + [[0, 0, 0]] * 2 and at == [0, 6, 6]


@pytest.mark.parametrize("page_size", [16, 24, 100, 1000])
def test_the_default_cache_serves_all_positions_and_no_more(page_size):
    """Pages that do not divide the model's 512 positions: a request gets all of them, and the next token is refused although its last page has room."""
    m = _model(1)
    cache = m.new_paged_cache(2, n_pages=80, page_size=page_size)
    assert cache.capacity == 512
    kv = m.new_cache(1, 511)
    kv.length = 511
    assert cache.fill(kv, [0]).status.tolist() == [0, 0]
    ids, ones = torch.tensor([3, 4], device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    for t, lengths, status in ((0, [512, 1], [0, 0]), (1, [512, 2], [2, 0])):
        logits = m.decode_paged(ids, cache, ones)
        assert cache.lengths.tolist() == lengths and cache.status.tolist() == status and logits[1].isfinite().all()
    check_status()


def test_a_cache_holds_as_many_tokens_as_it_was_made_for():
    m = _model(1)
    cache = m.new_paged_cache(1, n_pages=10, page_size=16, max_tokens=20)
    assert cache.capacity == 20
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    for t in range(22):
        m.decode_paged(torch.tensor([7], device="cuda"), cache, one)
        assert (cache.lengths.item(), cache.status.item()) == (min(t + 1, 20), 0 if t < 20 else 2)
    for page_size, max_tokens in ((16, -1), (0, 20)):
        with pytest.raises(ValueError):
            m.new_paged_cache(1, 10, page_size, max_tokens)


def test_what_is_refused_leaves_the_cache_as_it_was():
    """Tokens of another type or on the host, a cache or prompts of another model: no request grows by tokens whose keys were never written, no page is lost."""
    import decode_model as D
    m = _model(1)
    cache = m.new_paged_cache(2, 10, 16, 64)
    ones = torch.ones(2, dtype=torch.int32, device="cuda")
    ids = torch.tensor([3, 4], device="cuda")
    m.decode_paged(ids, cache, ones)
    deep, wide = _model(1, n_layers=3), _model(1, n_kv_heads=4)
    kv = lambda m: D.KVCache(*(m.new_cache(2, 64).k for _ in range(2)), length=16)
    calls = [lambda: m.decode_paged(ids.int(), cache, ones), lambda: m.decode_paged(ids.cpu(), cache, ones), lambda: deep.decode_paged(ids, cache, ones), lambda: wide.decode_paged(ids, cache, ones),
             lambda: cache.fill(kv(deep), [0, 1]), lambda: cache.fill(kv(wide), [0, 1]), lambda: cache.fill(D.KVCache(*(t.float() for t in (kv(m).k, kv(m).v)), length=16), [0, 1])]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
        assert cache.lengths.tolist() == [1, 1] and cache.n_free.item() == 8, i
    m.decode_paged(ids, cache, ones)
    assert cache.lengths.tolist() == [2, 2]


def test_a_step_of_a_batch_together():
    """Plan, decode, settings, sampling: the step of a server, for requests that each have settings of their own, against the plain formulas on the same logits."""
    import paged_cases as ref
    import seq_ops as S
    m = _model(2)
    B, g = 6, torch.Generator(device="cuda").manual_seed(1)
    cache = m.new_paged_cache(B, 40, 16, 96)
    said = torch.zeros(B, 64, dtype=torch.int64, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    ids = torch.arange(B, device="cuda") * 7
    new = torch.ones(B, dtype=torch.int32, device="cuda")
    rep, pres, freq = 1 + torch.rand(B, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
    mask = torch.randint(-2 ** 31, 2 ** 31, (B, 32), generator=g, device="cuda").int()
    prompt = torch.full((B,), 2, dtype=torch.int32, device="cuda")
    for t in range(20):
        said[:, t] = ids
        logits = m.decode_paged(ids, cache, new).float()
        kw = dict(tokens=said, lengths=cache.lengths, repetition=rep, presence=pres, frequency=freq, mask=mask)
        got = S.adjust_logits(logits, prompt_lengths=prompt, **kw)
        want, size = ref.adjust(logits, said, cache.lengths, prompt, rep, pres, freq, None, None, mask)
        off = torch.isinf(want)
        assert torch.equal(torch.isinf(got.cpu()), off) and ((got.double().cpu() - want).abs() <= 8 * 2.0 ** -24 * size)[~off].all()
        ids = S.sample(got, pos)
        assert torch.equal(ids, got.argmax(-1)) and not off[torch.arange(B), ids.cpu()].any()
        pos += 1
    assert cache.lengths.tolist() == [20] * B


def test_settings_of_a_request_in_the_engine():
    """Greedy generation with every setting, against the same steps by hand."""
    import paged_cases as ref
    from engine import Engine, SamplingParams
    m = _model(3)
    prompt = [5, 17, 17, 900, 3]
    plain = Engine(m, 64).generate([prompt], SamplingParams(max_new=12))[0]
    assert plain == Engine(m, 64).generate([prompt], SamplingParams(max_new=12, repetition=1.0, presence=0.0, frequency=0.0, bias=()))[0]
    word = lambda out: range(len(out) % 3, 1000, 3)
    params = SamplingParams(max_new=12, repetition=1.7, presence=0.4, frequency=0.3, bias=((11, 0.5), (11, 0.25), (600, -1.0)), allowed=word)
    got = Engine(m, 64).generate([prompt], params)[0]
    cache, tokens, out = m.new_cache(1, 64), list(prompt), []
    for _ in range(12):
        feed = tokens if not out else out[-1:]
        logits = m.forward(torch.tensor([feed]), cache, [len(feed) - 1])
        bits = torch.zeros(32 * 32, dtype=torch.int64)
        bits[list(word(out))] = 1
        mask = (bits.view(32, 32) << torch.arange(32)).sum(1)
        want, _ = ref.adjust(logits, torch.tensor([prompt + out]), [len(prompt) + len(out)], [len(prompt)], 1.7, 0.4, 0.3, torch.tensor([[11, 11, 600]]), torch.tensor([[0.5, 0.25, -1.0]]),
                             mask.view(1, -1))
        top = want[0].topk(2).values
        assert top[0] - top[1] > 1e-4          # no tie that a rounding decides
        out.append(int(want[0].argmax()))
    assert got == out and all(t % 3 == i % 3 for i, t in enumerate(got))
    eng = Engine(m, 64)
    with pytest.raises(ValueError):
        eng.submit(prompt, SamplingParams(repetition=0.0))
    with pytest.raises(ValueError):
        eng.submit(prompt, SamplingParams(bias=((1000, 1.0),)))
    with pytest.raises(ValueError):
        eng.generate([prompt], SamplingParams(allowed=lambda out: []))


def test_an_empty_cache_fills_nothing():
    m = _model(1)
    c = m.new_paged_cache(2, 10, 16, 64)
    p = c.fill(m.new_cache(2, 64), [0, 1])
    assert p.status.tolist() == [0, 0] and p.slots.numel() == 0 and c.lengths.tolist() == [0, 0] and c.n_free.item() == 10
    check_status()


def test_too_many_biases_are_refused_when_they_come():
    from engine import Engine, SamplingParams
    eng = Engine(_model(3), 64)
    with pytest.raises(ValueError):
        eng.submit([5, 17], SamplingParams(bias=((1, 0.5),) * 4097))
    assert not eng.waiting
    out = eng.generate([[5, 17]], SamplingParams(max_new=2, bias=((7, 0.125),) * 4096))[0]      # 512 in all
    assert out == [7, 7]


def test_a_request_that_fails_ends_alone():
    """No token allowed at the third: the request is gone, the other one gives what it gives by itself."""
    from engine import Engine, SamplingParams
    m = _model(3)
    want = Engine(m, 64).generate([[9, 4, 2]], SamplingParams(max_new=6))[0]
    eng = Engine(m, 64)
    bad = eng.submit([5, 17], SamplingParams(max_new=6, allowed=lambda out: range(1000) if len(out) < 2 else []))
    good = eng.submit([9, 4, 2], SamplingParams(max_new=6))
    with pytest.raises(ValueError):
        eng.run()
    assert eng.run()[good] == want and bad not in eng.finished and bad not in eng.pool


@pytest.mark.parametrize("words", [lambda: torch.tensor([7, 7]), lambda: torch.tensor([7, 7], device="cuda"), lambda: [7, 7],
                                   lambda: __import__("numpy").array([7, 7])], ids=["tensor", "device", "list", "array"])
def test_allowed_tokens_of_any_kind(words):
    """The same token several times is allowed once, whatever holds the numbers."""
    from engine import Engine, SamplingParams
    out = Engine(_model(3), 64).generate([[5, 17]], SamplingParams(max_new=6, allowed=lambda out: words()))[0]
    assert out == [7] * 6


def test_a_generation_that_fails_leaves_nothing_behind():
    """One of three prompts fails: none of them runs on in the next generation, none keeps a state or a result; the error names the request. Requests of others are untouched."""
    from engine import Engine, SamplingParams
    m = _model(3)
    want = Engine(m, 64).generate([[9, 4, 2], [8]], SamplingParams(max_new=4))
    eng = Engine(m, 64, max_live=2)
    other = eng.submit([9, 4, 2], SamplingParams(max_new=4))

    def fails(out):
        if len(out) == 2:
            raise KeyError("no rule")
    with pytest.raises(KeyError, match="no rule") as e:
        eng.generate([[5, 17], [6], [7, 7]], SamplingParams(max_new=6, allowed=fails))
    assert "2 tokens" in e.value.__notes__[0] and not eng.failed
    assert eng.generate([[8]], SamplingParams(max_new=4)) == want[1:]
    assert eng.finished == {other: want[0]} and not eng.live and not eng.waiting and not eng.pool.live
    with pytest.raises(ValueError):                # the second prompt is refused: the first one does not stay
        eng.generate([[5], []], SamplingParams(max_new=4))
    assert not eng.live and not eng.waiting and not eng.pool.live


def test_a_request_that_fails_is_recorded_and_stops_nobody_else():
    from engine import Engine, SamplingParams
    m = _model(3)
    want = Engine(m, 64).generate([[9, 4, 2], [8]], SamplingParams(max_new=4))
    eng = Engine(m, 64)
    bad = eng.submit([5, 17], SamplingParams(max_new=6, allowed=lambda out: range(1000) if len(out) < 2 else []))
    assert eng.generate([[9, 4, 2], [8]], SamplingParams(max_new=4)) == want       # whose request it is not
    error, tokens = eng.failed.pop(bad)
    assert isinstance(error, ValueError) and repr(bad) in error.__notes__[0] and len(tokens) == 2
    eng.submit([5, 17], SamplingParams(max_new=6, allowed=lambda out: []))
    assert eng.generate([], None) == [] and len(eng.failed) == 1
    gone = [eng.submit([5], SamplingParams(max_new=3)) for _ in range(2)]
    eng.run_one()
    for rid in gone + gone:
        eng.cancel(rid)
    assert not eng.live and not eng.waiting and not eng.pool.live and not eng.run()


def test_settings_from_the_command_line(tmp_path, capsys):
    import cli
    import model_registry as R
    m = _model(3)
    cfg = {"architecture": "PalettizedQwen", "max_positions": 512, **{k: getattr(m.cfg, k) for k in ("hidden", "n_heads", "n_kv_heads", "head_dim", "intermediate", "n_layers", "vocab")}}
    R.save_model(str(tmp_path), cfg, m.state_dict())
    run = lambda *a: (cli.main(["generate", "--model", str(tmp_path), "--tokens", "5,17,3", "--max-new", "6", *a]), list(map(int, capsys.readouterr().out.split())))
    assert run("--bias", "7:1000") == (0, [7] * 6)
    rc, out = run("--repetition", "1.5", "--presence", "1000", "--bias", "7:500")      # once said, a token is far away
    assert rc == 0 and out[0] == 7 and len(set(out)) == 6
