"""Models, the engine and the generator over a paged cache."""
import pytest
import torch

from summa_b200 import mal
from summa_b200.models import Transformer
from summa_b200.models.engine import InferenceEngine
from summa_b200.models.generate import SamplingConfig, TextGenerator
from summa_b200.models.paged import PagedCache

gpu = pytest.mark.gpu
KINDS = ["paged", "paged_e4m3"]


def _cfg(heads=4, kv=2, dim=64, extra="", layers=2):
    return mal.parse_mal(f"""
    attention a {{ num_heads: {heads} num_kv_heads: {kv} head_dim: {dim} bias: false {extra} }}
    ffn f {{ hidden_dim: 384 activation: swiglu bias: false }}
    block b {{ attention: a ffn: f norm: rmsnorm {{ eps: 1e-5 }} }}
    model m {{ vocab_size: 500 max_seq_len: 512 hidden_size: {heads * dim} num_layers: {layers} block: b }}
    """)


def _model(device, cfg=None, seed=0, std=0.08):
    torch.manual_seed(seed)
    with torch.device(device):
        m = Transformer(cfg or _cfg(), init_std=std)
    return m.prepare_inference(torch.bfloat16) if device == "cuda" else m.eval()


def _prompts(lengths, seed=1, vocab=500):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() if n else None for n in lengths]


# ------------------------------------------------------------------ the page table

def test_pages_are_taken_and_given_back():
    c = PagedCache(3, 100, page=16, num_pages=9)
    c.begin([17, 0, 48])
    assert c.held == [0, -1, 0] and [len(p) for p in c.pages] == [2, 0, 3] and len(c.free) == 4
    c.advance([17, 0, 48])
    assert c.lengths.tolist() == [17, -1, 48] == c.held
    used = sorted(c.pages[0] + c.pages[2])
    assert len(set(used)) == 5 and c.table[0, :2].tolist() == c.pages[0] and c.table[1].tolist() == [-1] * 7
    with pytest.raises(RuntimeError, match="overflow"):
        c.begin([0, 65, 16])                                     # six pages, four free
    assert [len(p) for p in c.pages] == [2, 0, 3] and c.held == [17, -1, 48]
    with pytest.raises(RuntimeError, match="capacity"):
        c.begin([84, 0, 0])
    c.release(2)
    assert c.held[2] == -1 and len(c.free) == 7 and c.table[2].tolist() == [-1] * 7 and c.lengths[2] == -1
    rows = c.begin([1, 65, 0])
    assert rows.starts.tolist() == [0, 1, 66, 66] and rows.max_rows == 65
    assert c.begin([1, 1, 1]).starts is None
    c.reset()
    assert c.held == [-1] * 3 and sorted(c.free) == list(range(9))
    for bad in ([1, 2], [1, -1, 0]):
        with pytest.raises(ValueError):
            c.begin(bad)
    with pytest.raises(ValueError):
        c.release(3)
    for args in ((0, 10), (1, 0), (1, 10, 24), (1, 10, 16, 0)):
        with pytest.raises(ValueError):
            PagedCache(*args)


# ------------------------------------------------------------------ models

@pytest.mark.parametrize("name", ["nano", "hybrid_tiny", "bench_tiny", "tiny"])
def test_paged_equals_contiguous_on_the_cpu(name):
    cfg = mal.get_builtin_model(name)
    cfg.vocab_size = 300
    torch.manual_seed(0)
    m = Transformer(cfg).eval()
    tok = torch.randint(0, 300, (2, 40))
    with torch.no_grad():
        a, b = m.make_state(2, 64), m.make_paged_state(2, 64, page=16)
        for i, j in ((0, 19), (19, 20), (20, 33), (33, 40)):
            x, y = m.forward_with_state(tok[:, i:j], a), m.forward_with_state(tok[:, i:j], b)
            torch.testing.assert_close(y, x, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("extra", ["", "qk_norm: true", "window_size: 20", "position_encoding: none", "causal: false"])
def test_ragged_prompts_equal_each_alone(extra):
    """Prompts of several lengths at once, a second part behind a history, a slot that joins later: logits as of each sequence alone."""
    m = _model("cpu", _cfg(extra=extra))
    first, second = _prompts([7, 33, 0, 1]), _prompts([0, 5, 21, 2], seed=2)
    st = m.make_paged_state(4, 128, page=16)
    with torch.no_grad():
        got = [m.forward_ragged_with_state(p, st) for p in (first, second)]
        for b in range(4):
            alone = m.make_state(1, 128)
            for part, logits in zip((first[b], second[b]), got):
                if part is None:
                    assert (logits[b] == 0).all()
                    continue
                want = m.forward_next_logits_with_state(torch.tensor([part]), alone)
                torch.testing.assert_close(logits[b:b + 1], want, rtol=1e-4, atol=1e-4)


def test_steps_pass_over_slots_that_are_not_in_use():
    m = _model("cpu")
    st = m.make_paged_state(3, 64, page=16)
    p = _prompts([9, 0, 4])
    with torch.no_grad():
        m.forward_ragged_with_state(p, st)
        pages = st.layers[0].kv.k.clone()
        m.forward_next_logits_with_state(torch.tensor([[1], [2], [3]]), st)
        assert st.paged.lengths.tolist() == [10, -1, 5] == st.paged.held
        assert (st.layers[0].kv.k != pages).any((1, 3)).sum() == 2           # one row in two pages
        with pytest.raises(ValueError):
            m.forward_with_state(torch.zeros(3, 2, dtype=torch.long), st)
        with pytest.raises(ValueError):
            m.forward_with_state(torch.zeros(2, 1, dtype=torch.long), st)


def test_released_sequences_leave_nothing_behind():
    """New prompts after all slots were released, in a model with recurrent layers: as in a fresh state."""
    cfg = mal.get_builtin_model("hybrid_tiny")
    cfg.vocab_size = 300
    torch.manual_seed(0)
    m = Transformer(cfg).eval()
    a, b = torch.randint(0, 300, (2, 2, 20))
    with torch.no_grad():
        st = m.make_paged_state(2, 64)
        m.forward_with_state(a, st)
        for slot in (0, 1):
            st.paged.release(slot)
        torch.testing.assert_close(m.forward_with_state(b, st), m.forward_with_state(b, m.make_paged_state(2, 64)), rtol=0, atol=0)


def test_a_prompt_is_one_row():
    m = _model("cpu")
    st = m.make_paged_state(2, 64)
    with pytest.raises(ValueError):
        m.forward_ragged_with_state([torch.ones(1, 5, dtype=torch.long), None], st)
    assert st.paged.held == [-1, -1] and len(st.paged.free) == st.paged.num_pages


def test_paged_refusals():
    m = _model("cpu")
    with pytest.raises(ValueError):
        m.make_paged_state(1, 600)                                           # max_seq_len 512
    with pytest.raises(ValueError):
        m.make_paged_state(1, 64, "int8")
    with pytest.raises(ValueError):
        m.forward_ragged_with_state([[1]], m.make_state(1, 8))
    st = m.make_paged_state(2, 64)
    with pytest.raises(ValueError):
        m.forward_ragged_with_state([[1]], st)
    cfg = mal.get_builtin_model("hybrid_tiny")
    cfg.vocab_size = 300
    h = Transformer(cfg).eval()
    with pytest.raises(ValueError, match="recurrent"):
        h.forward_ragged_with_state([[1], [2, 3]], h.make_paged_state(2, 64))
    eng = InferenceEngine(m)
    eng.reset(2, 64)
    for call in (lambda: eng.prefill_ragged([[1], [2]]), lambda: eng.release(0), lambda: eng.reset(1, 64, num_pages=4)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    eng.reset(2, 64, "paged")
    with pytest.raises(RuntimeError):
        eng.decode(torch.zeros(2, 1, dtype=torch.long), 1)


def test_a_state_of_ones_own_keeps_its_length():
    """Whatever has `k`, `v` and `length` is a contiguous state, not `AttentionState` alone."""
    from types import SimpleNamespace
    m = _model("cpu")
    tok = torch.randint(0, 500, (2, 30), generator=torch.Generator().manual_seed(0))
    with torch.no_grad():
        a, b = m.make_state(2, 64), m.make_state(2, 64)
        b.layers = [SimpleNamespace(k=st.k, v=st.v, length=0) for st in b.layers]
        for i, j in ((0, 12), (12, 13), (13, 30)):
            assert torch.equal(m.forward_with_state(tok[:, i:j], b), m.forward_with_state(tok[:, i:j], a))

# ------------------------------------------------------------------ engine and generator

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_generator_over_pages(device, kind):
    """Greedy tokens. On the CPU the pages hold what the contiguous cache does; in 8 bits and on the GPU the same run twice agrees, past the
    end of the cache too (the generator then brings the last half again)."""
    m = _model(device)
    prompt = _prompts([60])[0]
    cfg = SamplingConfig(max_new_tokens=20)
    out = TextGenerator(m, kv_cache=kind).generate_ids(prompt, cfg)
    assert out == TextGenerator(m, kv_cache=kind).generate_ids(prompt, cfg) and len(out) == 20
    if device == "cpu" and kind == "paged":
        assert out == TextGenerator(m).generate_ids(prompt, cfg)
    assert len(TextGenerator(m, kv_cache=kind).generate_ids(_prompts([505])[0], cfg)) == 20


def test_command_line_takes_the_cache(tmp_path, monkeypatch, capsys):
    from summa_b200.cli import llm
    seen = {}

    class Gen:
        def __init__(self, model, tok, kv_cache=None):
            seen["kv"] = kv_cache

        def generate(self, prompt, cfg):
            return prompt

    monkeypatch.setattr(llm, "_load", lambda args: (None, None, None))
    monkeypatch.setattr("summa_b200.models.generate.TextGenerator", Gen)
    base = ["generate", "--model", "m", "--tokenizer", "t", "--prompt", "p"]
    for more, want in (([], None), (["--kv-cache", "paged"], "paged"), (["--kv-cache", "paged_e4m3"], "paged_e4m3")):
        assert llm.main(base + more) == 0 and seen["kv"] == want
    with pytest.raises(SystemExit):
        llm.main(base + ["--kv-cache", "fp4"])


@torch.no_grad()
def _agrees(eng, seqs, prompts, kind, slack):
    """Every token of the captured decode is, but for rounding, what an eager pass over the same tokens picks."""
    eng.use_graph = False
    eng.reset(len(prompts), 400, kind)
    logits = eng.model.forward_ragged_with_state(prompts, eng.state).float()
    agree = 0
    for t in range(seqs.shape[1]):
        pick = seqs[:, t]
        gap = logits.max(-1).values - logits.gather(1, pick[:, None]).squeeze(1)
        assert float(gap.max()) < slack, (t, float(gap.max()))
        agree += int((logits.argmax(-1) == pick).sum())
        logits = eng.model.forward_next_logits_with_state(pick[:, None], eng.state).float()
    assert agree >= 0.9 * seqs.numel()


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim,extra,quantize", [(4, 2, 128, "", "int4"), (8, 2, 64, "qk_norm: true", None), (4, 4, 64, "window_size: 50", None)])
def test_captured_decode_of_ragged_sequences(heads, kv, dim, extra, quantize, kind):
    from summa_b200.ops import native
    cfg = _cfg(heads, kv, dim, extra)
    eng = InferenceEngine.build(cfg, torch.device("cuda"), quantize=quantize, init_std=0.05, seed=3)
    prompts = _prompts([200, 3, 77])
    outs = []
    for _ in range(2):
        eng.reset(3, 400, kind)
        first = eng.prefill_ragged(prompts)
        a = eng.decode(first, 10)
        outs.append(torch.cat([first, a, eng.decode(a[:, -1:], 10)], 1))
    assert eng._graph is not None and eng._graph.graph is not None and torch.equal(outs[0], outs[1])
    assert eng.state.paged.held == eng.state.paged.lengths.tolist() == [220, 23, 97]
    _agrees(eng, outs[0], prompts, kind, 0.15)
    assert native.read_error_flag() == 0


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_sequences_join_and_leave_while_others_go_on(kind):
    """A slot is released and taken by another prompt between captured steps: the sequences that go on are not disturbed, and the new one
    gets the tokens that it gets alone."""
    eng = InferenceEngine.build(_cfg(4, 2, 128), torch.device("cuda"), quantize=None, init_std=0.05, seed=4)
    a, b, c = _prompts([120, 31, 65], seed=7)
    eng.reset(2, 400, kind, num_pages=8)
    first = eng.prefill_ragged([a, b])
    x = eng.decode(first, 8)
    eng.release(1)
    new = eng.prefill_ragged([None, c])
    assert new[0, 0] == 0
    y = eng.decode(torch.stack([x[0, -1:], new[1]]), 8)
    assert eng.state.paged.held == [136, 73]
    with pytest.raises(RuntimeError, match="overflow"):
        eng.prefill_ragged([None, _prompts([390])[0]])
    eng.reset(2, 400, kind, num_pages=8)
    alone = eng.prefill_ragged([a, None])
    z = eng.decode(alone, 16)
    assert torch.equal(torch.cat([x[0], y[0]]), z[0])
    eng.reset(2, 400, kind, num_pages=8)
    alone = eng.prefill_ragged([None, c])
    assert torch.equal(alone[1], new[1]) and torch.equal(eng.decode(alone, 8)[1], y[1])


@gpu
@torch.no_grad()
def test_hybrid_and_equal_lengths_over_pages():
    """Recurrent and attention layers, prompts of one length: the captured steps over pages pick what the contiguous cache's do, but for
    rounding (attention of the contiguous steps rounds its weights to bf16 too)."""
    cfg = mal.get_builtin_model("hybrid_mamba_1536")
    cfg.num_layers, cfg.vocab_size = 6, 512
    eng = InferenceEngine.build(cfg, torch.device("cuda"), quantize=None, init_std=0.02, seed=1)
    tok = torch.randint(0, 512, (2, 50), generator=torch.Generator().manual_seed(2)).cuda()
    eng.reset(2, 128, "paged")
    first = eng.prefill(tok)
    out = torch.cat([first, eng.decode(first, 12)], 1)
    assert eng._graph is not None and eng._graph.graph is not None and eng.state.paged.held == [62, 62]
    eng.use_graph = False
    eng.reset(2, 128)
    logits = eng.model.forward_next_logits_with_state(tok, eng.state).float()
    for t in range(out.shape[1]):
        gap = logits.max(-1).values - logits.gather(1, out[:, t:t + 1]).squeeze(1)
        assert float(gap.max()) < 0.15, (t, float(gap.max()))
        logits = eng.model.forward_next_logits_with_state(out[:, t:t + 1], eng.state).float()


def _stamp(cache):
    return (list(cache.held), cache.lengths.tolist(), cache.table.tolist(), [list(p) for p in cache.pages], list(cache.free), cache.rows)


@pytest.mark.parametrize("kind", KINDS)
def test_a_pass_that_fails_leaves_the_slots_as_they_were(kind):
    """A token that is none, and a layer that raises: lengths, pages and slots in use are those of before, and what comes then is right."""
    m = _model("cpu")
    st, clean = (m.make_paged_state(3, 64, kind, page=16) for _ in range(2))
    first, second = _prompts([9, 0, 20]), _prompts([30, 5, 0], seed=2)
    with torch.no_grad():
        before = _stamp(st.paged)
        with pytest.raises(IndexError):
            m.forward_ragged_with_state([[1, 2], None, [3] * 40 + [10 ** 6]], st)
        assert _stamp(st.paged) == before
        assert torch.equal(m.forward_ragged_with_state(first, st), m.forward_ragged_with_state(first, clean))
        before = _stamp(st.paged)
        for call in (lambda: m.forward_ragged_with_state([[10 ** 6], [1], None], st),
                     lambda: m.forward_with_state(torch.tensor([[1], [2], [10 ** 6]]), st)):
            with pytest.raises(IndexError):
                call()
            assert _stamp(st.paged) == before
        assert torch.equal(m.forward_ragged_with_state(second, st), m.forward_ragged_with_state(second, clean))
        assert _stamp(st.paged) == _stamp(clean.paged)
        # behind the first layer: its rows are in the pages already, where nobody reads them (in 8 bits they may have moved a page's scale)
        before = _stamp(st.paged)
        hook = m.layers[1].register_forward_pre_hook(lambda *_: 1 // 0)
        with pytest.raises(ZeroDivisionError):
            m.forward_ragged_with_state(_prompts([3, 3, 14], seed=5), st)
        hook.remove()
        assert _stamp(st.paged) == before
        x, y = (m.forward_next_logits_with_state(torch.tensor([[4], [5], [6]]), s) for s in (st, clean))
        torch.testing.assert_close(x, y, rtol=0, atol=0 if kind == "paged" else 0.05 * float(y.abs().max()))


def test_a_pass_that_fails_leaves_recurrent_layers_as_they_were():
    cfg = mal.get_builtin_model("hybrid_tiny")
    cfg.vocab_size = 300
    torch.manual_seed(0)
    m = Transformer(cfg).eval()
    a, b = torch.randint(0, 300, (2, 2, 20))
    with torch.no_grad():
        st, clean = m.make_paged_state(2, 64), m.make_paged_state(2, 64)
        for tok in (a, b):
            hook = m.layers[-1].register_forward_pre_hook(lambda *_: 1 // 0)
            with pytest.raises(ZeroDivisionError):
                m.forward_with_state(tok, st)
            hook.remove()
            assert torch.equal(m.forward_with_state(tok, st), m.forward_with_state(tok, clean))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_a_captured_decode_that_fails_can_be_called_again(kind, monkeypatch):
    """The capture behind the first step raises: the lengths are those of before the call, and the same call then gives what it gives alone."""
    from summa_b200.models import engine
    eng = InferenceEngine.build(_cfg(4, 2, 128), torch.device("cuda"), quantize=None, init_std=0.05, seed=4)
    prompts = _prompts([60, 63], seed=3)
    eng.reset(2, 400, kind)
    want = eng.decode(eng.prefill_ragged(prompts), 8)
    eng.reset(2, 400, kind)
    eng._graph = None
    first = eng.prefill_ragged(prompts)
    before = _stamp(eng.state.paged)
    with monkeypatch.context() as mp:
        mp.setattr(engine._GraphDecoder, "_capture", lambda *_: 1 // 0)
        with pytest.raises(ZeroDivisionError):
            eng.decode(first, 8)
    assert _stamp(eng.state.paged) == before and eng.state.pos == 0
    assert torch.equal(eng.decode(first, 8), want)
    assert eng.state.paged.held == eng.state.paged.lengths.tolist() == [68, 71]
