"""The serving operators together, as a decoder uses them: a ragged prefill and decode
steps over the paged cache, products in 8-bit integers, captured, on other streams; and
the decoder's own ragged generation."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import pare_amd as P
from oracle import serving_oracle as S
from pare_amd.decoder import DecoderConfig, QuantizedDecoder, add_rmsnorm

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
CODES = [torch.int8, torch.float8_e4m3fn]
SMALL = DecoderConfig(hidden=1024, heads=8, kv_heads=2, ffn=2048, vocab=2000, layers=2)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _rope(L, D):
    a = np.arange(L)[:, None] / 10000.0 ** (np.arange(0, D, 2) / D)
    return (torch.from_numpy(f(a).astype(np.float32)).to(DEV) for f in (np.cos, np.sin))


def _against_64_bits(q, out, cache, layer, plan, scale):
    """Attention over the pages as they are read back, in 64 bits: half a step of fp16 in
    the output and in the probabilities, the latter twice (numerator and sum) with their
    scores' fp32 sums (2^-12), and the smallest subnormal's half."""
    pages = cache.k_scale[layer].shape[0]
    k, v = P.read_kv_pages(torch.arange(pages, dtype=torch.int32, device=DEV), cache.k[layer], cache.v[layer],
                           cache.k_scale[layer], cache.v_scale[layer], dtype=torch.float32)
    k, v = (t.double().cpu().numpy() for t in (k, v))
    o, weight = S.attention(q.double().cpu().numpy(), k, v, cache.block_tables.cpu().numpy(),
                            plan.kv_lens.cpu().numpy(), plan.q_starts.cpu().numpy(), cache.page_size, scale)
    err = np.abs(out.double().cpu().numpy() - o)
    assert (err <= 2.0 ** -11 * np.abs(o) + (2.0 ** -11 + 2.0 ** -12) * weight + 2.0 ** -25).all(), err.max()


class _Run:
    """Two layers' worth of a model's serving step on random activations."""

    def __init__(self, seed, requests, max_len, code, H=8, KV=2, D=128, page_size=32):
        g = torch.Generator().manual_seed(seed)
        self.g, self.R, self.H, self.KV, self.D = g, requests, H, KV, D
        self.cache = P.PagedKVCache(2, requests, max_len, KV, D, DEV, page_size=page_size, dtype=code)
        self.cos, self.sin = _rope(max_len, D)
        self.w, self.ws = P.quantize_rows(torch.randn(200, H * D, generator=g).to(DEV))
        self.max_len = max_len

    def draw(self, tokens):
        return torch.randn(2, tokens, (self.H + 2 * self.KV) * self.D, generator=self.g).half().to(DEV)

    def step(self, qkv, new_lens, max_q_len, check=False):
        plan = self.cache.extend(new_lens, qkv.shape[1])
        y = []
        for layer in range(2):
            q = self.cache.append(layer, qkv[layer], self.cos, self.sin, plan)
            o = self.cache.attend(layer, q, plan, scale=self.D ** -0.5, max_q_len=max_q_len)
            if check:
                _against_64_bits(q, o, self.cache, layer, plan, self.D ** -0.5)
            y.append(P.matmul_w8a8(o.reshape(o.shape[0], -1), self.w, self.ws))
        return torch.stack(y), plan

    def state(self):
        c = self.cache
        return [c.block_tables, c.kv_lens, c.pool, *c.k, *c.v, *c.k_scale, *c.v_scale]

    def copy(self, other):
        for a, b in zip(self.state(), other.state()):
            a.copy_(b)


def _equal(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a.state(), b.state()))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("D,page_size", [(128, 32), (64, 128)])
def test_prompts_then_steps_then_new_requests(code, D, page_size):
    """Prompts, decode steps, a request that ends and gives its pages to a longer one
    admitted in its place while the others go on."""
    run = _Run(1, 4, 700, code, D=D, page_size=page_size)
    new = [130, 1, 0, 300]
    run.step(run.draw(sum(new)), _ints(new), 300, check=True)
    one = _ints([1, 1, 0, 1])
    for _ in range(3):
        run.step(run.draw(3), one, 1, check=True)
    held = run.cache.pool[1].item()
    run.cache.release(torch.tensor([True, False, False, False], device=DEV))
    assert run.cache.kv_lens.tolist() == [0, 4, 0, 303]
    assert run.cache.pool[1].item() == held + -(-133 // page_size)
    new = [500, 1, 77, 1]
    run.step(run.draw(sum(new)), _ints(new), 500, check=True)
    assert run.cache.kv_lens.tolist() == [500, 5, 77, 304] and run.cache.pool[2].item() == 0


@pytest.mark.parametrize("code", CODES)
def test_captured_step_replays(code):
    """A captured step replayed many times, its twin run eagerly between the replays: the
    same cache and the same outputs, bit for bit, after each."""
    a, b = _Run(2, 3, 4200, code), _Run(2, 3, 4200, code)
    new = [4000, 1, 90]
    prompt = a.draw(sum(new))
    a.step(prompt, _ints(new), 4000)
    b.step(prompt, _ints(new), 4000)
    assert _equal(a, b)
    one, qkv = _ints([1, 1, 1]), a.draw(3)
    kept = _Run(2, 3, 4200, code)
    kept.copy(b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.step(qkv, one, 1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y, plan = b.step(qkv, one, 1)
    torch.cuda.current_stream().wait_stream(s)
    b.copy(kept)
    for i in range(40):
        qkv.copy_(a.draw(3))
        want, plan_a = a.step(qkv, one, 1, check=i == 0)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(y, want), f"replay {i}"
        assert torch.equal(plan.slots, plan_a.slots) and _equal(a, b), f"replay {i}"


def test_two_graphs_and_two_streams_at_once():
    """Captured steps of two caches replayed at the same time on two streams, and eager
    ones of a third between: nobody sees another's workspace."""
    runs = [_Run(3 + i, 2, 5000, torch.int8) for i in range(3)]
    twins = [_Run(3 + i, 2, 5000, torch.int8) for i in range(3)]
    new, one = _ints([4800, 33]), _ints([1, 1])
    inputs, graphs, outs = [], [], []
    streams = [torch.cuda.Stream() for _ in runs]
    for run, twin, s in zip(runs, twins, streams):
        prompt = run.draw(4833)
        run.step(prompt, new, 4800)
        twin.step(prompt, new, 4800)
        inputs.append(run.draw(2))
        s.wait_stream(torch.cuda.current_stream())
    for i in (0, 1):
        with torch.cuda.stream(streams[i]):
            twins[i].step(inputs[i], one, 1)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[i]):
                outs.append(twins[i].step(inputs[i], one, 1)[0])
            graphs.append(graph)
    torch.cuda.synchronize()
    for i in (0, 1):
        twins[i].copy(runs[i])
    torch.cuda.synchronize()
    for k in range(8):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            y = twins[2].step(inputs[2], one, 1)[0]
        torch.cuda.synchronize()
        want = [run.step(x, one, 1)[0] for run, x in zip(runs, inputs)]
        for i, got in enumerate([*outs, y]):
            assert torch.equal(got, want[i]) and _equal(runs[i], twins[i]), (k, i)


# --- the decoder ----------------------------------------------------------------------


@pytest.fixture(scope="module")
def model():
    return QuantizedDecoder(SMALL, DEV, seed=3)


def _prompts(lens, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, SMALL.vocab, (n,), generator=g).to(DEV) for n in lens]


@pytest.mark.parametrize("code", CODES)
def test_paged_layers_attend_to_their_own_requests(model, code, monkeypatch):
    """Every layer's attention of a ragged prefill and of the steps after it, against 64
    bits over what its pages hold; the first layer's pages against its own rotated keys."""
    cache = model.new_paged_cache(3, 100, page_size=16, dtype=code)
    cos, sin = model.rope_tables(100)
    seen = []
    attend = cache.attend
    monkeypatch.setattr(cache, "attend", lambda layer, q, plan, **kw: seen.append(layer) or _record(layer, q, plan, kw))

    def _record(layer, q, plan, kw):
        out = attend(layer, q, plan, **kw)
        _against_64_bits(q, out, cache, layer, plan, kw["scale"])
        return out

    prompts = _prompts([40, 1, 17])
    with torch.no_grad():
        plan = cache.extend(_ints([40, 1, 17]), 58)
        logits = model.forward_paged(torch.cat(prompts), cos, sin, cache, plan, max_q_len=40, max_kv_len=40)
        x = torch.nn.functional.embedding(torch.cat(prompts), model.embed)
        layer = model.layers[0]
        qkv = layer.qkv.fused(add_rmsnorm(x[None], None, layer.attn_norm.weight, SMALL.rms_eps)[0])[0]
        pos = plan.positions.cpu().numpy()
        assert pos.tolist() == [*range(40), 0, *range(17)]
        want = S.rotate(qkv.double().cpu().numpy().reshape(58, -1, 128)[:, 8:10], cos.double().cpu().numpy()[pos],
                        sin.double().cpu().numpy()[pos])
        got, _ = P.read_kv_pages(torch.arange(21, dtype=torch.int32, device=DEV), cache.k[0], cache.v[0],
                                 cache.k_scale[0], cache.v_scale[0], dtype=torch.float32)
        slots = plan.slots.cpu().numpy()
        got = got.double().cpu().numpy()[slots // 16, :, slots % 16]
        for page in set(slots // 16):
            a, b = got[slots // 16 == page], want[slots // 16 == page]
            top = np.abs(b).max((0, 2), keepdims=True)
            half = top / 254 if code == torch.int8 else np.maximum(np.abs(b) * 2.0 ** -4, top / 448 * 2.0 ** -10)
            assert (np.abs(a - b) <= half + top * 2.0 ** -20).all()
        for _ in range(3):
            plan = cache.extend(_ints([1, 1, 1]), 3)
            tokens = logits.argmax(-1)
            logits = model.forward_paged(tokens, cos, sin, cache, plan, max_q_len=1, max_kv_len=100)
    assert seen == [0, 1] * 4 and cache.kv_lens.tolist() == [43, 4, 20]
    assert logits.shape == (3, SMALL.vocab) and torch.isfinite(logits).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("lens", [[24], [5, 90, 1], [33] * 6])
def test_ragged_generation_graph_matches_eager(model, code, lens):
    prompts = _prompts(lens)
    eager, _ = model.generate_ragged(prompts, 20, dtype=code, use_graph=False)
    graph, t = model.generate_ragged(prompts, 20, dtype=code)
    again, _ = model.generate_ragged(prompts, 20, dtype=code)
    assert eager.shape == (len(lens), 20) and set(t) == {"prefill_s", "decode_s", "elapsed_s"}
    assert torch.equal(eager, graph) and torch.equal(graph, again)


def test_ragged_generation_ends_at_eos(model):
    """Until the first request ends, every call is the one made without eos; from then on
    the ended row is eos, and the others go on."""
    prompts = _prompts([20, 51, 7, 30])
    free, _ = model.generate_ragged(prompts, 16)
    eos = free[1, 6].item()
    first = min((row.tolist() + [eos]).index(eos) for row in free)
    for use_graph in (False, True):
        got, _ = model.generate_ragged(prompts, 16, eos=eos, use_graph=use_graph)
        assert torch.equal(got[:, :first + 1], free[:, :first + 1])
        for row in got.tolist():
            at = (row + [eos]).index(eos)
            assert row[at:] == [eos] * (16 - at)
        if use_graph:
            assert torch.equal(got, before)
        before = got


def test_one_token_and_refusals(model):
    prompts = _prompts([9, 2])
    assert torch.equal(model.generate_ragged(prompts, 1)[0], model.generate_ragged(prompts, 4)[0][:, :1])
    for bad in ([], [torch.zeros(0, dtype=torch.long)], [torch.zeros(1, 2, dtype=torch.long)]):
        with pytest.raises(ValueError):
            model.generate_ragged(bad, 4)
    with pytest.raises(ValueError):
        model.generate_ragged(prompts, 0)
    with pytest.raises(ValueError):
        model.generate_ragged(prompts, 4, dtype=torch.float16)


def test_int8_output_head():
    """Logits of the int8 head against the fp16 one's weight in 64 bits: each factor is off
    by at most half its code, sx and sw / 2 (and 2^-22 of the row's largest for the fp32
    division), and the result is rounded once to fp16."""
    model = QuantizedDecoder(SMALL, DEV, seed=7)
    w = model.lm_head.detach().double().cpu()
    before = model.linear_bytes_per_token()
    model.quantize_head()
    model.quantize_head()  # a second call changes nothing
    assert model.lm_head is None and before - model.linear_bytes_per_token() == 2000 * 1024 - 4 * 2000
    n = torch.randn(5, SMALL.hidden, generator=torch.Generator().manual_seed(1)).half()
    got = model._head(n.to(DEV)).double().cpu()
    x = n.double()
    dx = x.abs().amax(1, keepdim=True) * (1 / 254 + 2.0 ** -22)
    dw = w.abs().amax(1) * (1 / 254 + 2.0 ** -22)
    want = x @ w.T
    tol = x.abs().sum(1, keepdim=True) * dw + dx * w.abs().sum(1) + SMALL.hidden * dx * dw
    assert ((got - want).abs() <= tol * (1 + 2.0 ** -11) + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()
    out, _ = model.generate_ragged(_prompts([12, 3]), 6)
    again, _ = model.generate_ragged(_prompts([12, 3]), 6, use_graph=False)
    assert torch.equal(out, again)
    prompt = torch.stack(_prompts([12, 12]))
    assert torch.equal(model.generate(prompt, 6)[0], model.generate(prompt, 6, use_graph=False)[0])


def test_the_unfused_decoder_runs_with_an_int8_head_outside_no_grad():
    """Its plain ops record a graph up to the head, which has no backward pass."""
    model = QuantizedDecoder(SMALL, DEV, seed=7, fused_ops=False)
    model.quantize_head()
    cos, sin = model.rope_tables(8)
    tokens = torch.arange(8, device=DEV)[None]
    args = (tokens, cos, sin, model.new_cache(1, 8), torch.arange(8, device=DEV), None, True)
    with torch.no_grad():
        want = model.forward_tokens(*args)
    got = model.forward_tokens(*args)
    assert not got.requires_grad and torch.equal(got, want)


def test_a_decoder_with_an_int8_head_is_saved_and_loaded(tmp_path):
    model = QuantizedDecoder(SMALL, DEV, seed=7)
    model.quantize_head()
    prompts = _prompts([12, 3])
    want = model.generate_ragged(prompts, 6)[0]
    other = QuantizedDecoder(SMALL, DEV, seed=8)
    assert not torch.equal(other.generate_ragged(prompts, 6)[0], want)
    other.quantize_head()
    other.load_state_dict(model.state_dict())
    assert torch.equal(other.generate_ragged(prompts, 6)[0], want)
    with pytest.warns(UserWarning, match="8-bit"):
        P.save_quantized(model, tmp_path)
    third = P.load_quantized(QuantizedDecoder(SMALL, DEV, seed=9), tmp_path, device=DEV)
    assert torch.equal(third.generate_ragged(prompts, 6)[0], want)
