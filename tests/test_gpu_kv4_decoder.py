"""QuantDecoder with a 4-bit KV cache: prompts, decode steps and eviction.

The reference is the float64 decoder of test_gpu_decoder.py, whose attention takes the rows that
the decoder's own cache holds (read back): what the codes are is tested bit for bit in
test_gpu_kv4.py, so only the arithmetic around them remains, to the tolerance of that file's
float64 comparisons (1e-4 of the logits).
"""
import importlib

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_decoder import TINY, Reference, _rel  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec():
    return importlib.import_module("artifex-assistantv5_amd.decoder")


@pytest.fixture(scope="module")
def kv4(pkg):
    return importlib.import_module("artifex-assistantv5_amd.kv4")


def _model(dec, **over):
    cfg = dec.DecoderConfig(**{**TINY, **over})
    return cfg, dec.synthetic_weights(cfg, seed=3, device="cuda", distinct_layers=True)


class FromCache(Reference):
    """A Reference whose attention takes the given rows of each layer, [T, n_kv, hd]."""

    def token(self, tok, pos, rows):
        c = self.cfg
        x = self.embed[tok]
        nh, nkv, hd = c.n_heads, c.n_kv_heads, c.head_dim
        for (K, V), L in zip(rows, self.layers):
            qkv = L["qkv"] @ self.norm(x, L["an"])
            q = self.rope(qkv[:nh * hd].view(nh, hd), pos)
            heads = []
            for h in range(nh):
                kv = h // (nh // nkv)
                s = (K[:, kv] @ q[h]) / hd ** 0.5
                p = torch.exp(s - s.max())
                heads.append((p / p.sum()) @ V[:, kv])
            x = x + L["o"] @ torch.cat(heads)
            gu = L["gu"] @ self.norm(x, L["fn"])
            g, u = gu[:c.ffn], gu[c.ffn:]
            x = x + L["down"] @ (u * g / (1 + torch.exp(-g)))
        return self.lm @ self.norm(x, self.fnorm)


def _cached(kv4, m):
    """The cached rows of every layer, float64 [T, n_kv, hd]."""
    n = int(m.kv_lengths.item())
    shape = (*m.kv4.shape[:3], n, m.cfg.head_dim)
    k, v = (torch.zeros(shape, device="cuda") for _ in range(2))
    kv4.load(m.kv4, m.kv_lengths, k, v)
    return [(a[0].transpose(0, 1).double(), b[0].transpose(0, 1).double()) for a, b in zip(k, v)]


def _tokens(cfg, n, seed):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, cfg.vocab, n)).cuda()


@pytest.mark.parametrize("over", [{}, dict(n_heads=2, n_kv_heads=1, head_dim=128),
                                  dict(n_heads=8, n_kv_heads=1, head_dim=256)])
def test_prompt_and_steps(dec, kv4, over):
    cfg, w = _model(dec, **over)
    m = dec.QuantDecoder(cfg, w, kv_bits=4)
    exact = Reference(cfg, w)
    ref = FromCache(cfg, w)
    prompt = _tokens(cfg, 30, 5)
    logits = m.prefill(prompt, 0)[0]
    for p, t in enumerate(prompt.tolist()):
        rl = exact.token(t, p)
    assert _rel(logits, rl) < 1e-4           # one chunk: its rows attend in f32
    tok, pos = torch.argmax(logits).view(1), torch.tensor([30], device="cuda")
    for _ in range(4):
        t, p = int(tok.item()), int(pos.item())
        lg = m.step(tok, pos)[0]
        assert int(m.kv_lengths.item()) == p + 1
        assert _rel(lg, ref.token(t, p, _cached(kv4, m))) < 1e-4
    # a second prompt behind the steps: the last row attends to the cache and, in f32, its chunk
    more = _tokens(cfg, 7, 6)
    held = _cached(kv4, m)
    lg = m.prefill(more, 34)[0]
    assert int(m.kv_lengths.item()) == 41
    ref2 = Reference(cfg, w)
    ref2.k, ref2.v = [list(k) for k, _ in held], [list(v) for _, v in held]
    for i, t in enumerate(more.tolist()):
        rl = ref2.token(t, 34 + i)
    assert _rel(lg, rl) < 1e-4


def test_graph_matches_eager_with_eviction(dec):
    """Generation over a cache that fills up again and again; prompts longer than the cache."""
    cfg, w = _model(dec, max_seq=400)
    for prompt_len in (20, 150):
        prompt = _tokens(cfg, prompt_len, 7)
        outs = []
        for graph in (False, True):
            m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=64, kv_keep=40, kv_recent=16)
            outs.append(m.generate(prompt, 120, graph=graph)["tokens"])
            n = int(m.kv_lengths.item())
            assert 40 <= n < 64
            at = m.kv_positions[:, 0, :, :n]
            last = prompt_len + 119 - 1          # of the last token that was fed
            for row in at.reshape(-1, n).tolist():
                assert len(set(row)) == n and set(range(4)) <= set(row)
                assert set(range(last - 15, last + 1)) <= set(row) and max(row) == last
        assert torch.equal(*outs)


def test_eviction_keeps_what_fits(dec):
    """Until the cache is full nothing differs from a cache without eviction."""
    cfg, w = _model(dec, max_seq=128)
    prompt = _tokens(cfg, 30, 8)
    a = dec.QuantDecoder(cfg, w, kv_bits=4).generate(prompt, 30)["tokens"]
    b = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=96, kv_keep=48,
                         kv_recent=10).generate(prompt, 30)["tokens"]
    assert torch.equal(a, b)


def test_weights_of_a_prompt(dec, kv4):
    """After a prompt each slot holds the attention weight of the last rows: per layer and KV
    head they add up to one per row and query head."""
    cfg, w = _model(dec)
    m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=64, kv_keep=40, kv_recent=8)
    m.prefill(_tokens(cfg, 50, 9), 0)
    s = m.kv_weights[:, 0, :, :50].double().sum(-1)
    grp = cfg.n_heads // cfg.n_kv_heads
    assert torch.allclose(s, torch.full_like(s, 32.0 * grp), rtol=1e-5)


def test_refusals(dec):
    cfg, w = _model(dec)
    for bad in (dict(kv_bits=8), dict(kv_slots=64), dict(kv_keep=32), dict(kv_bits=4, fused=False),
                dict(kv_bits=4, hip_glue=False), dict(kv_bits=4, kv_slots=64, kv_keep=64),
                dict(kv_bits=4, kv_keep=20, kv_recent=17), dict(kv_bits=4, kv_slots=0)):
        with pytest.raises(ValueError):
            dec.QuantDecoder(cfg, w, **bad)
    m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=32)
    with pytest.raises(ValueError, match="slots"):
        m.prefill(_tokens(cfg, 33, 1), 0)
    with pytest.raises(ValueError, match="slots"):
        m.generate(_tokens(cfg, 20, 1), 20)


def test_a_prompt_follows_what_the_cache_holds(dec):
    cfg, w = _model(dec)
    tokens = _tokens(cfg, 12, 1)
    m = dec.QuantDecoder(cfg, w, kv_bits=4)
    whole = m.prefill(tokens, 0)
    m.prefill(tokens[:5], 0)
    for pos0 in (3, 7):
        with pytest.raises(ValueError, match="follow"):
            m.prefill(tokens[5:], pos0)
    # from position 5 on, over the first five rows as they are cached
    rest = m.prefill(tokens[5:], 5)
    assert int(m.kv_lengths.item()) == 12 and torch.isfinite(rest).all()
    m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=64, kv_keep=32, kv_recent=8)
    m.prefill(tokens[:5], 0)
    with pytest.raises(ValueError, match="follow"):
        m.prefill(tokens[5:], 4)
    assert whole.shape == rest.shape


def test_a_model_file_with_a_4_bit_cache(dec, tmp_path):
    """load_decoder passes the cache's form on: the tokens are those of the same decoder built
    directly, over an eviction, with RoPE frequency factors."""
    import gguf_models as gm

    gmodel = importlib.import_module("artifex-assistantv5_amd.gguf_model")
    tensors = gm.make_model(seed=6, rope_freqs=True)
    p = str(tmp_path / "m.gguf")
    gm.write_model(p, tensors)
    cache = dict(kv_bits=4, kv_slots=64, kv_keep=48, kv_recent=16)
    model, _ = gmodel.load_decoder(p, "cuda", max_seq=128, **cache)
    direct = dec.QuantDecoder(model.cfg, gm.direct_weights(tensors, gm.TINY), **cache)
    prompt = torch.from_numpy(np.random.default_rng(7).integers(0, model.cfg.vocab, 56)).cuda()
    a, b = model.generate(prompt, 30), direct.generate(prompt, 30, graph=False)
    assert torch.equal(a["tokens"], b["tokens"])
    assert int(model.kv_lengths.item()) == int(direct.kv_lengths.item()) < 64


def _state(m):
    return [t.clone() for t in m._cache_state()]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_prompt_that_does_not_fit_changes_nothing(dec):
    """Refused before the first layer, as with an f32 cache: the sequence goes on behind it."""
    cfg, w = _model(dec, max_seq=256)
    tokens = _tokens(cfg, 120, 3)
    m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=64)
    m.prefill(tokens[:40], 0)
    before = _state(m)
    for n, pos0 in ((25, 40), (65, 0), (120, 0)):
        with pytest.raises(ValueError, match="slots"):
            m.prefill(tokens[:n], pos0)
        assert _same(_state(m), before)
    got = m.prefill(tokens[40:64], 40)
    assert int(m.kv_lengths.item()) == 64 and torch.isfinite(got).all()


@pytest.mark.parametrize("cache", [{}, dict(kv_slots=64, kv_keep=32, kv_recent=8)])
def test_an_empty_prompt_is_refused(dec, cache):
    cfg, w = _model(dec)
    tokens = _tokens(cfg, 10, 3)
    m = dec.QuantDecoder(cfg, w, kv_bits=4, **cache)
    m.prefill(tokens, 0)
    before = _state(m)
    for pos0 in (0, 10):
        with pytest.raises(ValueError, match="empty"):
            m.prefill(tokens[:0], pos0)
        assert _same(_state(m), before)


def test_nothing_kept_is_refused(dec):
    cfg, w = _model(dec)
    for keep in (0, -1):
        with pytest.raises(ValueError, match="kv_keep"):
            dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=64, kv_keep=keep, kv_recent=0, kv_sinks=0)


@pytest.mark.parametrize("graph", [False, True])
def test_a_step_past_the_last_slot_is_seen(dec, graph):
    """Its logits are NaN, nothing is stored, and the cache still holds what it held."""
    cfg, w = _model(dec, max_seq=256)
    m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=32)
    prompt = _tokens(cfg, 29, 4)
    tok = torch.argmax(m.prefill(prompt, 0), dim=-1).view(1)
    pos = torch.tensor([29], device="cuda")
    if graph:
        m.capture(tok, pos)

    def step():
        if not graph:
            return m.step(tok, pos)
        m._graph.replay()
        return m._graph_logits

    for _ in range(3):
        assert torch.isfinite(step()).all()
    before = _state(m)
    for _ in range(3):
        assert torch.isnan(step()).all()
        assert _same(_state(m), before) and m.kv_lengths.tolist() == [32]
    with pytest.raises(ValueError, match="slots"):
        m.prefill(prompt[:1], 32)
    again = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=32)
    assert torch.equal(m.prefill(prompt, 0), again.prefill(prompt, 0))
    tok.fill_(7)
    pos.fill_(29)
    got = step().clone()
    tok.fill_(7)
    pos.fill_(29)
    assert torch.equal(got, again.step(tok, pos))


def test_a_step_past_the_tables_is_seen(dec):
    """With eviction the positions end with the RoPE tables."""
    cfg, w = _model(dec)
    m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=64, kv_keep=32, kv_recent=8)
    m.prefill(_tokens(cfg, 20, 4), 0)
    tok, pos = torch.tensor([1], device="cuda"), torch.tensor([m.cos.shape[0]], device="cuda")
    m.step(tok.clone(), torch.tensor([20], device="cuda"))
    assert torch.isnan(m.step(tok, pos)).all()


def test_a_prompt_follows_the_last_position(dec):
    """With eviction the slots in use do not tell the next position: one too far or one that was
    there already is refused, after prompts, steps and evictions, and what is held stays."""
    cfg, w = _model(dec, max_seq=400)
    tokens = _tokens(cfg, 200, 1)
    m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=64, kv_keep=32, kv_recent=0, kv_sinks=0)

    def refuses(*positions):
        before = _state(m)
        for p in positions:
            with pytest.raises(ValueError, match="follow"):
                m.prefill(tokens[:3], p)
        assert _same(_state(m), before)

    m.prefill(tokens[:5], 0)
    refuses(4, 6, 64)
    m.prefill(tokens[5:20], 5)
    refuses(5, 19, 21)
    m.prefill(tokens[20:150], 20)                     # over evictions
    assert int(m.kv_lengths.item()) < 64
    refuses(63, 149, 151, 200)
    tok, pos = tokens[150:151].clone(), torch.tensor([150], device="cuda")
    for _ in range(40):                               # and again
        m.step(tok, pos)
    refuses(150, 189, 191)
    m.prefill(tokens[:1], 190)
    out = m.generate(tokens[:50], 30)["tokens"]       # 79 tokens fed
    assert out.numel() == 30
    refuses(78, 80)
    m.prefill(tokens[:2], 79)


def test_prompts_of_any_length_share_a_workspace(dec):
    """Prompts of 1 .. 40 rows leave no more memory in use than the first did."""
    cfg, w = _model(dec, max_seq=2000)
    tokens = _tokens(cfg, 40, 2)
    warm = dec.QuantDecoder(cfg, w, kv_bits=4)        # what the projections keep is there
    for n in range(1, 41):
        warm.prefill(tokens[:n], 0)
    m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=1024, kv_keep=512)
    used, at = [], 0
    for n in (1, 40, 2, 33, 7, 32, 31, 5):
        m.prefill(tokens[:n], at)
        at += n
        torch.cuda.synchronize()
        used.append(torch.cuda.memory_allocated())
    assert used == used[:1] * len(used)


@pytest.mark.parametrize("over", [{}, dict(n_heads=8, n_kv_heads=1, head_dim=128)])
def test_prompt_and_steps_behind_evictions(dec, kv4, over):
    """Slots are out of order and behind the positions: a prompt's logits and those of steps are
    float64's over the rows that the cache holds."""
    cfg, w = _model(dec, max_seq=400, **over)
    tokens = _tokens(cfg, 320, 2)
    m = dec.QuantDecoder(cfg, w, kv_bits=4, kv_slots=64, kv_keep=40, kv_recent=16)
    ref = FromCache(cfg, w)
    m.prefill(tokens[:150], 0)
    held, at = _cached(kv4, m), 150
    assert m.kv_positions[0, 0, 0, :held[0][0].shape[0]].tolist() != list(range(held[0][0].shape[0]))
    for turn in range(3):
        n = min(9, 63 - held[0][0].shape[0])          # no eviction within
        lg = m.prefill(tokens[at:at + n], at)[0]
        exact = Reference(cfg, w)
        exact.k, exact.v = [list(k) for k, _ in held], [list(v) for _, v in held]
        for i in range(n):
            rl = exact.token(int(tokens[at + i]), at + i)
        assert _rel(lg, rl) < 1e-4
        at += n
        tok, pos = torch.argmax(lg).view(1), torch.tensor([at], device="cuda")
        for _ in range(40):                           # through an eviction
            t, p, before = int(tok.item()), int(pos.item()), int(m.kv_lengths.item())
            lg = m.step(tok, pos)[0]
            if before < 63:                           # else the rows attended to were cut
                assert int(m.kv_lengths.item()) == before + 1
                assert _rel(lg, ref.token(t, p, _cached(kv4, m))) < 1e-4
            at += 1
        held = _cached(kv4, m)
