"""Processed logits and greedy tokens against a plain implementation in 64 bits
(oracle/sharing_oracle.py): penalties, biases, masks, refusals, capture, streams."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import pare_amd as P
from oracle import sharing_oracle as O
from pare_amd import _lib

gpu = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float16, torch.bfloat16, torch.float32]
P8 = 0x1000  # an aligned address that is never read: validation comes first


def _case(R, V, L, n_bias, masks, dtype, seed=0, repeat=True):
    """Arguments as CPU tensors; tokens outside the vocabulary among them."""
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    a = dict(logits=(4 * torch.randn(R, V, generator=g)).to(dtype), history=None, history_lens=None, prompt_lens=None,
             repetition=None, presence=None, frequency=None, bias_ids=None, bias=None, allowed=None, allowed_rows=None)
    if L is not None:
        h = (V * rand(R, L) ** (4 if repeat else 1)).int()
        h[rand(R, L) < 0.02] = -1
        h[rand(R, L) < 0.02] = V
        a.update(history=h, history_lens=torch.randint(-1, L + 3, (R,), generator=g).int(),
                 prompt_lens=torch.randint(-1, L + 3, (R,), generator=g).int(), repetition=0.7 + rand(R),
                 presence=2 * rand(R) - 0.5, frequency=rand(R) - 0.2)
    if n_bias:
        ids = torch.randint(-2, V + 2, (R, n_bias), generator=g).int()
        if n_bias > 3:
            ids[:, 1] = ids[:, 3]  # a token with two biases
        a.update(bias_ids=ids, bias=5 * torch.randn(R, n_bias, generator=g))
    if masks:
        words = -(-V // 32)
        m = torch.randint(-2 ** 31, 2 ** 31, (masks, words), generator=g).int()
        m[0] = 0  # allows nothing
        a.update(allowed=m, allowed_rows=torch.randint(-1, masks + 1, (R,), generator=g).int())
    return a


def _on(a, dev=DEV):
    return {k: v.to(dev) if v is not None else None for k, v in a.items()}


def _want(a):
    n = {k: v.numpy() if v is not None and k != "logits" else v for k, v in a.items()}
    return O.logits(a["logits"].double().numpy(), *[n[k] for k in (
        "history", "history_lens", "prompt_lens", "repetition", "presence", "frequency", "bias_ids", "bias", "allowed",
        "allowed_rows")])


def _check(got, a):
    """Half a step of the type in the result. On the way fp32's half steps (2^-24), of the sum of the
    magnitudes each: a quotient or product, the frequency's product and two differences, the biases' sum
    (at most four of a token here) and its addition: eight."""
    want, size = _want(a)
    t = a["logits"].dtype
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[t]
    x = got.double().cpu().numpy()
    hidden = np.isneginf(want)
    assert (np.isneginf(x) == hidden).all()
    tol = torch.finfo(t).eps / 2 * np.abs(want[~hidden]) + 9 * 2.0 ** -24 * size[~hidden] + least
    err = np.abs(x[~hidden] - want[~hidden])
    assert (err <= tol).all(), (err - tol).max()


def _first_largest(x):
    """The lowest index of the largest value of each row."""
    return np.argmax(x.double().cpu().numpy(), 1)


# --- the oracle, refusals (CPU) ---------------------------------------------------------

def test_oracle_by_hand():
    x = np.array([[2.0, -2.0, 4.0, 1.0]])
    out, _ = O.logits(x, np.array([[0, 1, 1, 9, 0]]), np.array([4]), np.array([1]), np.array([2.0]), np.array([0.5]),
                      np.array([0.25]), np.array([[3, 3, -1]]), np.array([[1.0, 2.0, 7.0]]),
                      np.array([[0b1011]], np.int32), None)
    # token 0: only in the prompt; 1: twice behind it; 2 is not allowed; 3: two biases
    assert out.tolist() == [[1.0, -4.0 - 0.5 - 0.5, -np.inf, 4.0]]


def _args(greedy=False, **kw):
    a = dict(x=P8, dtype=_lib.PMI_F16, stride=100, history=P8, hstride=8, L=8, hlens=P8, plens=P8, rep=P8, pres=P8,
             freq=P8, ids=P8, bias=P8, n_bias=3, allowed=P8, masks=2, words=4, rows=P8)
    a.update(dict(tokens=P8, tstride=1) if greedy else dict(out=P8, ostride=100))
    a.update(R=2, V=100)
    if greedy:
        a.update(ws=P8, ws_bytes=1 << 40)
    a.update(kw)
    return [*a.values(), None]


BOTH = [dict(dtype=_lib.PMI_I8), dict(R=-1), dict(V=-1), dict(stride=99), dict(L=-1), dict(hstride=7), dict(n_bias=-1),
        dict(masks=-1), dict(x=None), dict(x=P8 + 1), dict(ids=None), dict(bias=None), dict(words=3),
        dict(rows=None, masks=1), dict(V=1 << 30, stride=1 << 30), dict(R=1 << 30), dict(L=1 << 31, hstride=1 << 31)]


@pytest.mark.parametrize("change", BOTH + [dict(out=None), dict(out=P8 + 1), dict(ostride=99)])
def test_process_logits_refuses(change):
    assert _lib.lib().pmi_process_logits(*_args(**change)) in (_lib.PMI_ERR_INVALID, _lib.PMI_ERR_UNSUPPORTED)


@pytest.mark.parametrize("change", [dict(out=P8 + 2), dict(out=P8 - 2), dict(out=P8 + 398), dict(out=P8 - 398),
                                    dict(ostride=101), dict(out=P8 + 200, ostride=101), dict(out=P8 + 2, R=1),
                                    dict(out=P8 + 198, stride=201, ostride=201), dict(out=P8 + 204, stride=201, ostride=201)])
def test_an_output_that_overlaps_the_logits_is_refused(change):
    assert _lib.lib().pmi_process_logits(*_args(**change)) == _lib.PMI_ERR_INVALID


@pytest.mark.parametrize("change", BOTH + [dict(tokens=None), dict(tstride=0), dict(V=0, words=0), dict(R=16385), dict(ws=None),
                                           dict(ws=P8 + 16), dict(ws_bytes=100)])
def test_greedy_tokens_refuses(change):
    assert _lib.lib().pmi_greedy_tokens(*_args(True, **change)) in (_lib.PMI_ERR_INVALID, _lib.PMI_ERR_UNSUPPORTED)


def test_empty_calls_do_nothing():
    L = _lib.lib()
    assert L.pmi_process_logits(*_args(R=0, x=None, out=None)) == _lib.PMI_OK
    assert L.pmi_process_logits(*_args(V=0, x=None, out=None)) == _lib.PMI_OK
    assert L.pmi_greedy_tokens(*_args(True, R=0, tokens=None, ws=None)) == _lib.PMI_OK


def test_cpu_tensors_raise():
    for call in (P.process_logits, P.greedy_tokens):
        with pytest.raises(RuntimeError):
            call(torch.zeros(1, 4))


@gpu
def test_python_checks():
    x = torch.zeros(2, 64, device=DEV)
    ints, floats = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(2, device=DEV)
    h = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    for call in (P.process_logits, P.greedy_tokens):
        for kw in (dict(repetition=floats), dict(history_lens=ints), dict(prompt_lens=ints),
                   dict(history=h.long()), dict(history=h[:1]), dict(history=h, presence=floats.half()),
                   dict(history=h, frequency=floats[:1]), dict(history=h, history_lens=ints.long()),
                   dict(bias_ids=h), dict(bias_ids=h, bias=floats), dict(bias=floats), dict(allowed=h),
                   dict(allowed=h[:1, :2]), dict(allowed_rows=ints), dict(allowed=h[:, :2].contiguous().long()),
                   dict(history=h.t().contiguous().t())):
            with pytest.raises(AssertionError):
                call(x, **kw)
        for y in (x.double(), x[0], x.t(), x[:, ::2], x[:1].expand(2, 64)):
            with pytest.raises(AssertionError):
                call(y)
        with pytest.raises(RuntimeError):
            call(x, history=h.cpu())
        with pytest.raises(RuntimeError):
            call(x, history=h, repetition=floats.cpu())
    for out in (x.half(), x[:1]):
        with pytest.raises(AssertionError):
            P.process_logits(x, out=out)
    for out in (ints, ints.long()[:1], torch.zeros(1, dtype=torch.int64, device=DEV).expand(2)):
        with pytest.raises(AssertionError):
            P.greedy_tokens(x, out=out)


# --- values -----------------------------------------------------------------------------

SIZES = [(1, 1, 1, 1, 1), (3, 31, 5, 4, 2), (2, 33, 0, 0, 1), (5, 4095, 40, 7, 3), (4, 4097, 300, 30, 2),
         (7, 8209, 1000, 0, 0), (3, 32000, 2000, 1500, 4), (2, 50257, None, 5, 2), (2, 5000, None, 0, 0)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,L,n_bias,masks", SIZES)
def test_against_64_bits(R, V, L, n_bias, masks, dtype):
    a = _case(R, V, L, n_bias, masks, dtype, seed=V)
    if n_bias > 100:  # few tokens with more than three biases; none here
        a["bias_ids"] = torch.stack([torch.randperm(V, generator=torch.Generator().manual_seed(r))[:n_bias].int()
                                     for r in range(R)])
    d = _on(a)
    got = P.process_logits(**d)
    _check(got, a)
    assert torch.equal(P.process_logits(**d), got)
    assert P.greedy_tokens(**d).tolist() == _first_largest(got).tolist()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_biases_of_one_token_are_added_in_their_order(dtype):
    """Bits of the sum, one fp32 addition after another, however many there are."""
    R, V, n = 2, 9000, 700
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 5, (R, n), generator=g).int() * 2000
    bias = torch.randn(R, n, generator=g)
    got = P.process_logits(torch.zeros(R, V, dtype=dtype, device=DEV), bias_ids=ids.to(DEV), bias=bias.to(DEV))
    want = np.zeros((R, V), np.float32)
    for r in range(R):
        for t in range(0, 10000, 2000):
            total = None
            for b in bias[r][ids[r] == t].numpy():
                total = b if total is None else np.float32(total + b)
            if t < V and total is not None:
                want[r, t] = total
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(dtype))


@gpu
def test_counts_of_long_histories():
    """One token 70000 times, among others; counts and the prompt's flag do not meet."""
    V, L = 5000, 70003
    h = torch.full((2, L), 4321, dtype=torch.int32)
    h[:, 70000:] = torch.tensor([1, 2, 1])
    a = dict(_case(2, V, None, 0, 0, torch.float32), history=h, prompt_lens=torch.tensor([0, 70001]).int(),
             repetition=torch.tensor([1.5, 1.5]), frequency=torch.tensor([0.25, 0.25]),
             presence=torch.tensor([1.0, 1.0]))
    got = P.process_logits(**_on(a))
    _check(got, a)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,stride,offset", [(1000, 1001, 0), (1001, 1003, 1), (4096, 4099, 5), (999, 1000, 7), (5, 64, 3)])
def test_rows_that_are_not_aligned(dtype, V, stride, offset):
    """Any stride and start, into an output of another one, in place as well; what lies around the
    rows stays."""
    R = 5
    a = _case(R, V, 60, 6, 2, dtype, seed=stride)
    d = _on(a)
    want = P.process_logits(**d)
    _check(want, a)
    room = torch.full((R * stride + 64,), 7.0, dtype=dtype, device=DEV)
    view = room[offset:offset + R * stride].view(R, stride)[:, :V]
    view.copy_(d["logits"])
    assert torch.equal(P.process_logits(**dict(d, logits=view)), want)
    assert P.greedy_tokens(**dict(d, logits=view)).tolist() == P.greedy_tokens(**d).tolist()
    other = torch.full((R * (stride + 1) + 64,), 7.0, dtype=dtype, device=DEV)
    to = other[1:1 + R * (stride + 1)].view(R, stride + 1)[:, :V]
    assert P.process_logits(**dict(d, logits=view), out=to) is to and torch.equal(to, want)
    assert P.process_logits(**dict(d, logits=view), out=view) is view and torch.equal(view, want)
    for buffer, t in ((room, view), (other, to)):
        t.fill_(7.0)
        assert (buffer == 7).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan(dtype):
    """Hidden ones leave no trace; the others go the way of the formula."""
    V = 200
    x = torch.zeros(4, V, dtype=dtype)
    x[0, 3], x[0, 5], x[0, 7], x[1, 100], x[1, 50] = float("nan"), float("inf"), -float("inf"), float("nan"), 9
    x[2] = -float("inf")
    x[3, 9:12] = torch.finfo(dtype).min
    h = torch.tensor([[3, 5, 7, 0]] * 4).int()
    mask = torch.full((2, 7), -1).int()
    mask[1, 0] = ~(1 << 3 | 1 << 5)
    kw = dict(history=h.to(DEV), repetition=torch.full((4,), 2.0, device=DEV), presence=torch.full((4,), 1.0, device=DEV),
              allowed=mask.to(DEV), allowed_rows=torch.tensor([1, 0, 0, 0]).int().to(DEV))
    got = P.process_logits(x.to(DEV), **kw).cpu()
    assert got[0, 3] == got[0, 5] == got[0, 7] == -float("inf") and torch.isfinite(got[0, 8:]).all()
    assert got[1, 100] != got[1, 100] and got[1, 50] == 9 and (got[2] == -float("inf")).all()
    assert (got[3, 9:12] == torch.finfo(dtype).min).all() and got[3, 5] == -1
    assert P.greedy_tokens(x.to(DEV), **kw).tolist() == [1, 100, 0, 1]
    free = P.process_logits(x.to(DEV), history=kw["history"], repetition=kw["repetition"]).cpu()
    assert free[0, 3] != free[0, 3] and free[0, 5] == float("inf") and free[0, 7] == -float("inf")
    assert P.greedy_tokens(x.to(DEV)).tolist()[:3] == [3, 100, 0]


@gpu
def test_greedy_ties_and_masks_that_allow_nothing():
    V = 20000
    x = torch.zeros(3, V, dtype=torch.float16, device=DEV)
    x[1, [19999, 8191, 8192, 12000]] = 3
    allowed = torch.zeros(2, V // 32, dtype=torch.int32, device=DEV)
    allowed[1, 12000 // 32] = 1 << (12000 % 32)
    allowed[1, 19999 // 32] = -2 ** 31  # bit 31
    assert P.greedy_tokens(x).tolist() == [0, 8191, 0]
    rows = torch.tensor([0, 1, 1], dtype=torch.int32, device=DEV)
    assert P.greedy_tokens(x, allowed=allowed, allowed_rows=rows).tolist() == [0, 12000, 12000]
    buffer = torch.full((3, 2), -5, dtype=torch.int64, device=DEV)
    assert P.greedy_tokens(x, out=buffer[:, :1]) is not None
    assert buffer.tolist() == [[0, -5], [8191, -5], [0, -5]]


@gpu
def test_neutral_arguments_change_nothing():
    x = torch.randn(3, 5003, device=DEV).to(torch.bfloat16)
    h = torch.arange(9, dtype=torch.int32, device=DEV).repeat(3, 1)
    ones, zeros = torch.ones(3, device=DEV), torch.zeros(3, device=DEV)
    for kw in (dict(), dict(history=h), dict(history=h, repetition=ones, presence=zeros, frequency=zeros),
               dict(history=h[:, :0], repetition=2 * ones), dict(bias_ids=h[:, :0], bias=x.float()[:, :0].contiguous()),
               dict(bias_ids=torch.full_like(h, -1), bias=torch.ones(3, 9, device=DEV)),
               dict(allowed=torch.zeros(1, 157, dtype=torch.int32, device=DEV),
                    allowed_rows=torch.tensor([-1, 1, 7], dtype=torch.int32, device=DEV))):
        assert torch.equal(P.process_logits(x, **kw), x)
    assert P.process_logits(x[:0]).shape == (0, 5003) and P.greedy_tokens(x[:0]).shape == (0,)
    assert P.process_logits(x[:, :0]).shape == (3, 0)


@gpu
def test_captured_and_on_other_streams():
    a = _on(_case(6, 12345, 200, 9, 3, torch.float16))
    first = P.process_logits(**a), P.greedy_tokens(**a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            out, tokens = P.process_logits(**a), P.greedy_tokens(**a)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        a["logits"].normal_(0, 4)
        a["history_lens"].fill_(40 * i)
        want = P.process_logits(**a), P.greedy_tokens(**a)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(tokens, want[1])
        assert not torch.equal(want[0], first[0])


@gpu
def test_no_call_waits_for_the_device():
    a = _on(_case(2, 3000, 20, 3, 2, torch.float16))
    P.greedy_tokens(**a)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        P.process_logits(**a)
        P.greedy_tokens(**a)
    finally:
        torch.cuda.set_sync_debug_mode("default")


@gpu
def test_logits_past_2_31_values():
    R, V = 16384, 140001
    x = torch.zeros(R, V, dtype=torch.bfloat16, device=DEV)
    at = torch.arange(R, device=DEV) * 7 % V
    x[torch.arange(R, device=DEV), at] = 5
    h = at.int()[:, None].contiguous()
    assert torch.equal(P.greedy_tokens(x), at)
    got = P.greedy_tokens(x, history=h, presence=torch.full((R,), 6.0, device=DEV))
    assert torch.equal(got, (at == 0).long())
    P.process_logits(x, history=h, presence=torch.full((R,), 6.0, device=DEV), out=x)
    assert (x.gather(1, at[:, None]) == -1).all() and int((x != 0).sum()) == R


@gpu
def test_an_output_beside_the_logits():
    """Halves of one buffer, and rows behind the logits' rows."""
    x = torch.randn(4, 100, device=DEV)
    want = P.process_logits(x)
    both = torch.cat([x, x * 0], 1)
    P.process_logits(both[:, :100], out=both[:, 100:])
    assert torch.equal(both[:, 100:], want) and torch.equal(both[:, :100], x)
    rows = torch.cat([x, x * 0])
    P.process_logits(rows[:4], out=rows[4:])
    assert torch.equal(rows[4:], want) and torch.equal(rows[:4], x)
    one = torch.cat([x[0], x[0] * 0]).view(1, 200)
    P.process_logits(one[:, :100], out=one[:, 100:])
    assert torch.equal(one[0, 100:], want[0])


@gpu
def test_a_gradient_is_refused():
    x = torch.zeros(2, 64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="backward"):
        P.process_logits(x)
    with torch.no_grad():
        assert not P.process_logits(x).requires_grad
    assert P.greedy_tokens(x).tolist() == [0, 0]


@gpu
@pytest.mark.parametrize("rows", [1000, 16384])
def test_many_rows(rows):
    x = torch.randn(rows, 4100, device=DEV)
    got = P.greedy_tokens(x)
    assert torch.equal(got, x.argmax(1))
    if rows == 16384:
        with pytest.raises(_lib.PmiError):
            P.greedy_tokens(torch.zeros(rows + 1, 8, device=DEV))


# --- limits of a launch ---------------------------------------------------------------------

@pytest.mark.parametrize("L", [1 << 30, (1 << 31) - 4096, (1 << 31) - 1])
def test_histories_past_2_30_are_refused(L):
    """The kernel goes through a history in steps of 4096 tokens with a 32-bit index: in one of more than 2^31 - 4096 it
    would go negative, and read before the row."""
    change = dict(L=L, hstride=L)
    assert _lib.lib().pmi_process_logits(*_args(**change)) == _lib.PMI_ERR_UNSUPPORTED
    assert _lib.lib().pmi_greedy_tokens(*_args(True, **change)) == _lib.PMI_ERR_UNSUPPORTED


@pytest.mark.parametrize("change", [dict(L=1 << 15, hstride=1 << 15), dict(n_bias=(1 << 16) - 1)])
def test_more_rows_than_a_launch_of_the_wide_form_holds_are_refused(change):
    """2^23 workgroups of 512 threads are 2^32 threads: the library's refusal, not the runtime's error."""
    for rows in (1 << 23, 1 << 31):
        assert _lib.lib().pmi_process_logits(*_args(R=rows, **change)) == _lib.PMI_ERR_UNSUPPORTED


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_past_a_launch_of_large_slices(dtype):
    """Rows that are workgroups enough take 1024 threads each, up to 2^22 of them; more are done in the form of 256.
    One fp32 sum and its rounding: the same bits."""
    for R in ((1 << 22) - 1, 1 << 22, (1 << 22) + 3):
        g = torch.Generator(device=DEV).manual_seed(R)
        x = torch.randn(R, 5, generator=g, device=DEV).to(dtype)
        at = torch.randint(0, 5, (R, 1), generator=g, device=DEV)
        value = torch.randn(R, 1, generator=g, device=DEV)
        got = P.process_logits(x, bias_ids=at.int(), bias=value)
        assert torch.equal(got, x.float().scatter_add(1, at, value).to(dtype))


# --- derivatives ------------------------------------------------------------------------------

def _float_arguments(dev):
    a = dict(logits=torch.zeros(2, 64), history=torch.zeros(2, 3, dtype=torch.int32), repetition=torch.ones(2),
             presence=torch.ones(2), frequency=torch.ones(2), bias_ids=torch.zeros(2, 3, dtype=torch.int32),
             bias=torch.ones(2, 3), out=torch.zeros(2, 64))
    return {k: v.to(dev) for k, v in a.items()}


DERIVED = ["logits", "repetition", "presence", "frequency", "bias", "out"]


def _refuses_derivatives(name, dev):
    a = _float_arguments(dev)
    a[name].requires_grad_()
    with pytest.raises(RuntimeError, match="backward"):
        P.process_logits(**a)
    a = _float_arguments(dev)
    with torch.autograd.forward_ad.dual_level():
        a[name] = torch.autograd.forward_ad.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            P.process_logits(**a)


@pytest.mark.parametrize("name", DERIVED)
def test_a_derivative_that_would_be_left_out_is_refused(name):
    _refuses_derivatives(name, "cpu")


@gpu
@pytest.mark.parametrize("name", DERIVED)
def test_a_derivative_of_any_argument_is_refused(name):
    """On the way through the host extension too; without a derivative, and for tokens, the call is done."""
    _refuses_derivatives(name, DEV)
    a = _float_arguments(DEV)
    want = P.process_logits(**a).clone()
    a[name].requires_grad_()
    with torch.no_grad():
        assert torch.equal(P.process_logits(**a), want)
    a = _float_arguments(DEV)
    with torch.autograd.forward_ad.dual_level():
        assert torch.equal(P.process_logits(**a), want)
    if name != "out":
        del a["out"]
        a[name].requires_grad_()
        assert P.greedy_tokens(**a).tolist() == [1, 1]


# --- the forms that large batches, long histories and many biases take ---------------------------

def _laid_out(x, stride):
    """x with rows `stride` values apart."""
    room = torch.zeros(x.shape[0], stride, dtype=x.dtype, device=x.device)
    return room[:, :x.shape[1]].copy_(x)


def _check_forms(a, strides):
    """Logits of several strides, written and in place, and their tokens."""
    d = _on(a)
    first = None
    for stride in strides:
        x = _laid_out(d["logits"], stride)
        got = P.process_logits(**dict(d, logits=x))
        if first is None:
            first = got
            _check(got, a)
            tokens = _first_largest(got).tolist()
        assert torch.equal(got, first)
        assert P.greedy_tokens(**dict(d, logits=x)).tolist() == tokens
        assert P.process_logits(**dict(d, logits=x), out=x) is x and torch.equal(x, first)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V", [(64, 70001), (300, 1003)])
def test_rows_that_are_workgroups_enough(R, V, dtype):
    """Slices of 16384 tokens: histories with prompts, repeated biases and masks; rows that are aligned, and that are not."""
    _check_forms(_case(R, V, 300, 30, 4, dtype, seed=R), (V, V + 8 - V % 8, V + 3))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [3, 40])
def test_long_histories_with_biases_and_masks(R, dtype):
    """Counts in 32 bits, in slices of 8192 tokens."""
    V = 20001
    a = _case(R, V, 40000, 30, 2, dtype, seed=R)
    a["history_lens"][0], a["prompt_lens"][0] = 40000, 39000
    a["history_lens"][1], a["prompt_lens"][1] = 33000, 0
    _check_forms(a, (V, V + 7, V + 2))


@gpu
@pytest.mark.parametrize("R", [2, 64])
@pytest.mark.parametrize("L", [(1 << 15) - 1, 1 << 15])
def test_one_token_that_fills_its_history(L, R):
    """The most that 16 bits with the prompt's flag count, and one more."""
    V, token = 70001, 65537
    h = torch.full((R, L), token, dtype=torch.int32)
    a = dict(_case(R, V, None, 5, 2, torch.float32, seed=L), history=h, prompt_lens=torch.arange(R).int() % 2,
             repetition=torch.full((R,), 1.5), frequency=torch.full((R,), 0.25), presence=torch.full((R,), 1.0))
    a["allowed"][1, token // 32] |= 1 << (token % 32)
    a["allowed_rows"][:2] = 1
    _check_forms(a, (V, V + 3))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [2, 64])
@pytest.mark.parametrize("n", [(1 << 16) - 2, (1 << 16) - 1])
def test_as_many_biases_as_16_bits_name_and_more(n, R, dtype):
    """The last entry of each form; a token with a first and a last bias, and none with more."""
    V = 70001
    a = _case(R, V, 20, 0, 1, dtype, seed=n)
    rows = [torch.randperm(V, generator=torch.Generator().manual_seed(r))[:n].int() for r in range(2)]
    ids = torch.stack([rows[r % 2] for r in range(R)])
    ids[0, n - 1] = ids[0, 0]
    a.update(bias_ids=ids, bias=5 * torch.randn(R, n, generator=torch.Generator().manual_seed(n)))
    _check_forms(a, (V,))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,n", [(2, 9000, 700), (64, 70001, 3000), (2, 70001, (1 << 16) + 50)])
def test_tokens_with_one_bias_beside_those_with_several(R, V, n, dtype):
    """Bits of the sums in the entries' order, in each form: every third entry is of a token that has another one."""
    g = torch.Generator().manual_seed(n)
    ids = torch.stack([torch.randperm(V, generator=g)[torch.arange(n) % V].int() for _ in range(2)])
    few = torch.randint(0, n // 5, ids[:, ::3].shape, generator=g)
    ids[:, ::3] = ids.gather(1, few - few % 3 + 1)
    bias = torch.randn(2, n, generator=g)
    pick = torch.arange(R) % 2
    x = torch.zeros(R, V, dtype=dtype, device=DEV)
    got = P.process_logits(x, bias_ids=ids[pick].to(DEV), bias=bias[pick].to(DEV))
    want = np.zeros((2, V), np.float32)
    for r in range(2):
        seen = set()
        for t, b in zip(ids[r].tolist(), bias[r].numpy()):
            want[r, t] = np.float32(want[r, t] + b) if t in seen else b
            seen.add(t)
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(dtype)[pick])
    tokens = P.greedy_tokens(x, bias_ids=ids[pick].to(DEV), bias=bias[pick].to(DEV))
    assert tokens.tolist() == _first_largest(got).tolist()
