"""Models on a paged cache: projections, rotation, pages, attention and the rest of a block as a server calls them, against the contiguous cache."""
import ctypes as C

import numpy as np
import pytest

from denograd_amd import ffi, synthetic
from denograd_amd.ffi import check
from denograd_amd.llama3 import Llama3
from denograd_amd.paged import PagedCache
from denograd_amd.tensor import Tensor
from tests.helpers import quantize_state

pytestmark = pytest.mark.gpu


def model(quantize="float16", **more):
    cfg = synthetic.config("tiny16", quantize=quantize, max_context=256, **more)
    sd = synthetic.random_state_dict(cfg, seed=3, std=0.05)
    return cfg, Llama3.from_config(cfg).load_weights(quantize_state(cfg, sd), quantized=True)


def cache_for(llm, n_pages=64, page_size=16, dtype="float16"):
    m = llm.model
    return PagedCache(len(m.layers), m.n_kv_heads, m.dim // m.n_heads, n_pages, page_size, dtype)


def logits(m, n):
    return m._paged.logits.numpy()[:n].astype(np.float64)


@pytest.mark.parametrize("quantize", ["float16", "int8", "nf4"])
def test_ragged_batches_give_the_logits_of_one_sequence_at_a_time(hip, quantize):
    """fp16 pages hold what the contiguous cache holds; the float sums of products and attention come in another order, so activations differ by roundings:
    the tolerance that the whole-model tests have for those (1e-2 of the largest logit)."""
    cfg, llm = model(quantize)
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, cfg["vocab_size"], n).astype(np.int32) for n in (5, 40, 1, 97)]
    more = rng.integers(0, cfg["vocab_size"], (4, 3)).astype(np.int32)
    want = []
    for p, t in zip(prompts, more):
        llm.model.forward_rows(p[None], 0)
        steps = [llm.model.logits.numpy().astype(np.float64)]
        for i, tok in enumerate(t):
            llm.model.forward_rows(np.array([[tok]], np.int32), p.size + i)
            steps.append(llm.model.logits.numpy().astype(np.float64))
        want.append(steps)
    cache = cache_for(llm)
    seqs = [cache.add() for _ in prompts]
    got = [[] for _ in prompts]
    llm.model.forward_paged(cache, seqs[:2], prompts[:2])
    for b, x in zip((0, 1), logits(llm.model, 2)):
        got[b].append(x)
    # two prompts join two running sequences
    llm.model.forward_paged(cache, [seqs[2], seqs[0], seqs[3], seqs[1]], [prompts[2], more[0, :1], prompts[3], more[1, :1]])
    for b, x in zip((2, 0, 3, 1), logits(llm.model, 4)):
        got[b].append(x)
    for i in (0, 1, 2):
        todo = [b for b in range(4) if i + (b < 2) < 3]
        tok = llm.model.forward_paged(cache, [seqs[b] for b in todo], [more[b, i + (b < 2):i + (b < 2) + 1] for b in todo])
        x = logits(llm.model, len(todo))
        assert np.array_equal(tok.numpy(), x.argmax(-1))
        for b, row in zip(todo, x):
            got[b].append(row)
    for g, w in zip(got, want):
        assert len(g) == len(w) == 4
        for x, y in zip(g, w):
            assert np.max(np.abs(x - y)) <= 1e-2 * np.abs(y).max()


@pytest.mark.parametrize("dtype", ["float16", "int8"])
def test_a_prompt_in_one_piece_and_in_several(hip, dtype):
    """A position's codes and scales do not depend on what comes with it, so the pieces end in the logits of the whole."""
    cfg, llm = model()
    prompt = np.random.default_rng(1).integers(0, cfg["vocab_size"], 150).astype(np.int32)
    last = []
    for cuts in ((150,), (64, 149, 150), (1, 2, 33, 120, 150)):
        cache = cache_for(llm, dtype=dtype)
        s, at = cache.add(), 0
        for c in cuts:
            llm.model.forward_paged(cache, [s], [prompt[at:c]])
            at = c
        last.append(logits(llm.model, 1)[0])
    for x in last[1:]:
        assert np.max(np.abs(x - last[0])) <= 1e-2 * np.abs(last[0]).max()


def test_generate_paged_and_pages_given_away_behind_a_window(hip):
    """A sequence with a window and sinks goes on the same whether its old pages are given away or kept."""
    cfg, llm = model()
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, cfg["vocab_size"], n).astype(np.int32) for n in (70, 3, 33)]
    plain = llm.generate_paged(prompts, 5)
    assert plain.shape == (3, 5) and plain.dtype == np.int32
    assert np.array_equal(plain, llm.generate_paged(prompts, 5, page_size=128))
    assert llm.generate_paged(prompts, 2, dtype="int8").shape == (3, 2)
    keep, give = cache_for(llm, 40), cache_for(llm, 40)
    sk, sg = [keep.add() for _ in prompts], [give.add() for _ in prompts]
    toks, given = prompts, 0
    for _ in range(30):
        a = llm.model.forward_paged(keep, sk, toks, 24, 2).numpy()
        x = logits(llm.model, 3)
        b = llm.model.forward_paged(give, sg, toks, 24, 2).numpy()
        assert np.array_equal(a, b) and np.array_equal(x, logits(llm.model, 3))
        given += sum(give.slide(s, 24, 2) for s in sg)
        toks = list(a)
    # lengths 99, 32 and 62 in the end, so that positions from 76, 9 and 39 on are seen: pages 1 to 3 of the first, 1 of the last (page 0 has the sinks)
    assert given == 4 and len(give.free) == len(keep.free) + 4
    for s in sg:
        give.drop(s)
    assert sorted(give.free) == list(range(40))


def test_calls_that_are_refused_change_nothing(hip):
    cfg, llm = model()
    cache = cache_for(llm, 4)
    s = cache.add()
    ok = np.arange(10, dtype=np.int32)
    for bad, err in ((dict(tokens=[np.zeros(0, np.int32)]), ValueError), (dict(tokens=[np.array([cfg["vocab_size"]])]), ValueError), (dict(tokens=[ok, ok]), ValueError),
                     (dict(tokens=[np.zeros(65, np.int32)]), MemoryError), (dict(tokens=[np.zeros(513, np.int32)]), ValueError), (dict(seqs=[s, s], tokens=[ok, ok]), ValueError)):
        with pytest.raises(err):
            llm.model.forward_paged(cache, bad.get("seqs", [s]), bad["tokens"])
        assert cache.lengths[s] == 0 and len(cache.free) == 4
    with pytest.raises(ValueError, match="layers"):
        llm.model.forward_paged(PagedCache(1, 2, 64, 4), [0], [ok])
    batch = cache.begin([s], [10])
    k = Tensor.zeros((10, 2, 64), "float16")
    batch.write(0, k, k)
    with pytest.raises(ValueError, match="float16 rows"):
        batch.write(0, Tensor.zeros((9, 2, 64), "float16"), k)
    with pytest.raises(ffi.HipError, match="window"):
        batch.attend(0, Tensor.zeros((10, 4, 64), "float16"), 4, window=-1)
    cache.begin([s], [1])
    with pytest.raises(RuntimeError, match="another batch"):
        batch.read(0)


def test_an_attention_of_the_callers_own_takes_its_rows_normed(hip):
    """As with several rows (TransformerBlock.call_rows).  The norm's squares are added in another order then: the tolerance of the whole-model tests."""
    _, llm = model()
    prompts = [np.arange(n, dtype=np.int32) for n in (9, 1, 30)]
    def run():
        cache = cache_for(llm)
        seqs = [cache.add() for _ in prompts]
        llm.model.forward_paged(cache, seqs, prompts)
        return logits(llm.model, 3)
    want, seen = run(), []
    for layer in llm.model.layers:
        def own(xn, *args, attention=layer.attention, norm=layer.attention_norm):
            seen.append((xn, norm))
            return type(attention).call_paged(attention, xn, *args)
        layer.attention.call_paged = own
    got = run()
    assert len(seen) == len(llm.model.layers) and all(x is llm.model._paged.xn for x, _ in seen)
    assert np.max(np.abs(got - want)) <= 1e-2 * np.abs(want).max()


def test_windows_and_sinks_below_zero_are_refused_in_front_of_the_first_layer(hip):
    _, llm = model()
    cache = cache_for(llm, 4)
    s = cache.add()
    for more in (dict(window=-1), dict(sinks=-1)):
        with pytest.raises(ValueError, match="window"):
            llm.model.forward_paged(cache, [s], [np.arange(3, dtype=np.int32)], **more)
        assert cache.lengths[s] == 0 and len(cache.free) == 4


def test_captured_calls_replay_with_what_the_arrays_hold_then(hip):
    """Write and attention of one step recorded once; lengths move on between the replays, with eager calls of another batch on the same workspace between."""
    rng = np.random.default_rng(5)
    H, KV, hd, page = 8, 2, 64, 16
    from tests.paged_ref import Case
    for kind in ("float16", "int8"):
        c, e = (Case(np.random.default_rng(6), kind, hd, KV, page, [1, 1, 1], [300, 40, 1000]).device() for _ in range(2))
        other = Case(rng, kind, hd, KV, page, [90, 1], [500, 700]).device()
        ws = Tensor.zeros((hip.jsgrad_hip_attn_paged_workspace_bytes(H, KV, hd),), "uint8")
        q, k, v, q2 = (Tensor(rng.standard_normal((n, h, hd)).astype(np.float16)) for n, h in ((3, H), (3, KV), (3, KV), (91, H)))
        out, ref, out2 = Tensor.zeros((3, H, hd), "float16"), Tensor.zeros((3, H, hd), "float16"), Tensor.zeros((91, H, hd), "float16")

        def step(case, to):
            check(hip.jsgrad_hip_paged_write(*case.batch, None, k.ptr, v.ptr, None, 0, None, 0))
            check(hip.jsgrad_hip_attn_paged(*case.batch, q.ptr, to.ptr, H, 0, 0, ws.ptr))

        graph = C.c_void_p()
        check(hip.jsgrad_hip_graph_begin())
        try:
            step(c, out)
        finally:
            check(hip.jsgrad_hip_graph_end(C.byref(graph)))
        for lens in ([100, 7, 900], [101, 8, 901], [33, 1, 64], [300, 40, 1000], [1, 16, 17]):
            for case in (c, e):
                case.t["lens"].lazydata.copyin(np.array(lens, np.int32))
            check(hip.jsgrad_hip_graph_launch(graph))
            got = out.numpy()
            check(hip.jsgrad_hip_attn_paged(*other.batch, q2.ptr, out2.ptr, H, 0, 0, ws.ptr))
            step(e, ref)
            assert np.array_equal(got, ref.numpy()) and got.any()
            assert np.array_equal(c.t["k"].numpy(), e.t["k"].numpy())
        check(hip.jsgrad_hip_graph_destroy(graph))
