"""The operators of the verify step together, as a decode step uses them: residual + norm -> e4m3 rows -> head
product -> draft verification (VerifyHead), behind a stack of layers (DecodeStack.verify)."""
import numpy as np
import pytest
import torch

import synth
from verify_oracle import verify

pytestmark = pytest.mark.gpu


def head_weights(V, hs, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    # rows of different lengths: peaked logits from a normalised input
    w = torch.randn(V, hs, generator=g, device="cuda") * hs ** -0.5 * (0.5 + 3.0 * torch.rand(V, 1, generator=g, device="cuda"))
    return (torch.randn(hs, generator=g, device="cuda") * 0.1 + 1.0).bfloat16(), w.bfloat16()


def drafts(logits, B, n, seed, noise=0.5):
    """What a drafter with an error of its own would have proposed for these rows."""
    V = logits.shape[1]
    g = torch.Generator(device="cuda").manual_seed(seed)
    guess = logits.view(B, n + 1, V)[:, :n].float()
    guess = (guess + noise * torch.randn(guess.shape, generator=g, device="cuda")).bfloat16()
    ids = torch.multinomial(torch.softmax(guess.float().view(B * n, V), 1), 1, generator=g).view(B, n).int()
    return ids, guess.reshape(B * n, V).contiguous(), torch.rand(B, n + 1, generator=g, device="cuda")


def expected(logits, ids, u, dl, T, lens, B, n):
    V = logits.shape[1]
    host = lambda t: None if t is None else t.float().cpu().numpy()
    d = None if dl is None else host(dl).reshape(B, n, V)
    return verify(host(logits).reshape(B, n + 1, V), ids.cpu().numpy(), u.cpu().numpy(), d, None if T is None else host(T),
                  None if lens is None else lens.cpu().numpy())


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("B,n,hs,V", [(1, 1, 256, 517), (4, 3, 512, 3001), (8, 3, 2048, 8192), (3, 7, 1040, 1000)])
def test_head(q4t, gpu_lib, B, n, hs, V, fp8):
    T = B * (n + 1)
    nw, w = head_weights(V, hs, V)
    head = q4t.VerifyHead(nw, w, B, n, fp8=fp8)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (2 * torch.randn(T, hs, generator=g, device="cuda")).bfloat16()
    y = torch.randn(T, hs, generator=g, device="cuda").bfloat16()
    r = (x.float() + y.float()).bfloat16()
    v = r.double() / (r.double().square().mean(1, keepdim=True) + 1e-6).sqrt() * nw.double()
    ids = torch.zeros(B, n, dtype=torch.int32, device="cuda")
    u = torch.rand(B, n + 1, generator=g, device="cuda")
    keep = x.clone()
    head(x, ids, u, y=y)
    assert torch.equal(x, r) and not torch.equal(x, keep)
    # logits against the formula: an e4m3 step (2^-4 of a value at most) of each operand in quadrature over the row
    # and a bf16 step of the result; bf16 operands: a bf16 step (2^-8) of the normalised input likewise
    want = v @ w.double().t()
    step = (2 * 2.0 ** -4 if fp8 else 2.0 ** -8)
    S2 = (v.square() @ w.double().square().t()).sqrt()
    assert ((head.logits.double() - want).abs() <= 8 * step * S2 + 2.0 ** -8 * want.abs()).all()
    # the tokens are those that the definition gives for these logits
    ids, dl, u = drafts(head.logits, B, n, 11)
    temp = 0.5 + torch.rand(B, generator=g, device="cuda")
    lens = torch.randint(0, n + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    for d, t, ln in ((dl, temp, None), (None, None, lens), (dl, temp, lens)):
        got = head(x, ids, u, draft_logits=d, temperature=t, draft_len=ln)
        tokens, accepted, probs, am, dm = expected(head.logits, ids, u, d, t, ln, B, n)
        assert am > 2.0 ** -18 and dm > 1e-12
        assert np.array_equal(got["tokens"].cpu().numpy(), tokens)
        assert np.array_equal(got["accepted"].cpu().numpy(), accepted)


def test_stack_with_verification(q4t, gpu_lib):
    """A whole step equals its parts, eagerly and as one CUDA graph replayed on other inputs."""
    E, hs, is_, sis, k, B, n, V, nl = 32, 512, 256, 128, 4, 6, 3, 2050, 3
    T = B * (n + 1)
    dls = [q4t.DeviceLayer.from_host(synth.make_layer(E=E, hs=hs, moe_is=is_, shared_is=sis, seed=90 + i)) for i in range(nl)]
    stack = q4t.DecodeStack(dls, T, k)
    nw, w = head_weights(V, hs, 1)
    head = q4t.VerifyHead(nw, w, B, n)
    g = torch.Generator(device="cuda").manual_seed(4)
    xs = [torch.randn(T, hs, generator=g, device="cuda").bfloat16() for _ in range(2)]
    greedy = torch.zeros(B, device="cuda")
    results = []
    for i, x0 in enumerate(xs):
        # the parts
        x = x0.clone()
        stack(x)
        codes = torch.empty(T, hs, dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.empty(T, device="cuda")
        q4t.residual_rmsnorm_fp8(x, None, nw, codes, scales)
        hc, hsc = q4t.quantize_rows_fp8(w)
        logits = q4t.linear(codes, hc, x_scale=scales, w_scale=hsc)
        ids, dl, u = drafts(logits, B, n, 20 + i)
        # greedy drafts of half the sequences are what the target says
        best = logits.view(B, n + 1, V)[:, :n].argmax(2).int()
        ids[::2] = best[::2]
        want = q4t.VerifyDrafts(B, n, V)(logits, ids, u, draft_logits=dl)
        want_greedy = q4t.VerifyDrafts(B, n, V)(logits, ids, u, temperature=greedy)
        # the step
        y = x0.clone()
        got = stack.verify(y, head, ids, u, draft_logits=dl)
        assert torch.equal(y, x) and torch.equal(head.logits, logits)
        assert all(torch.equal(got[key], want[key]) for key in want)
        got = stack.verify(x0.clone(), head, ids, u, temperature=greedy)
        assert all(torch.equal(got[key], want_greedy[key]) for key in want_greedy)
        assert (got["accepted"][::2] == n).all()
        results.append((ids, dl, u, want))
    x, ids, dl, u = xs[0].clone(), *[t.clone() for t in results[0][:3]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = stack.verify(x, head, ids, u, draft_logits=dl)
    for x0, (i2, d2, u2, want) in list(zip(xs, results))[::-1]:
        x.copy_(x0), ids.copy_(i2), dl.copy_(d2), u.copy_(u2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[key], want[key]) for key in want)
    q4t.linear_status()


def test_two_heads_on_two_threads(q4t, gpu_lib):
    """Two host threads drive one GPU, each with its own head and stream."""
    import threading
    nw, w = head_weights(4099, 512, 5)
    B, n = 4, 3
    heads = [q4t.VerifyHead(nw, w, B, n, fp8=f) for f in (True, False)]
    xs = [torch.randn(B * (n + 1), 512, device="cuda").bfloat16() for _ in heads]
    u = torch.rand(B, n + 1, device="cuda")
    want, args = [], []
    for h, x in zip(heads, xs):
        h(x, torch.zeros(B, n, dtype=torch.int32, device="cuda"), u)
        ids, dl, uu = drafts(h.logits, B, n, 2)
        args.append((ids, uu, dl))
        want.append(h(x, ids, uu, draft_logits=dl))
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        ids, uu, dl = args[i]
        for _ in range(20):
            got = heads[i](xs[i], ids, uu, draft_logits=dl, stream=s)
            s.synchronize()
            if not all(torch.equal(got[k], want[i][k]) for k in got):
                bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_row_counts_must_agree(q4t, gpu_lib):
    dl = q4t.DeviceLayer.from_host(synth.make_layer(E=8, hs=256, moe_is=128, shared_is=128, seed=1))
    nw, w = head_weights(100, 256, 5)
    stack, head = q4t.DecodeStack([dl], 8, 2), q4t.VerifyHead(nw, w, 2, 2)
    x = torch.zeros(8, 256, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(q4t.Q4TError, match="6 rows, the stack 8"):
        stack.verify(x, head, torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, device="cuda"))
    with pytest.raises(q4t.Q4TError, match="shape"):
        head(x, torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, device="cuda"))


FIRST_CALL = """
import sys
sys.path.insert(0, %r)
import importlib
import torch
q4t = importlib.import_module("qwen4-thor_b200")
torch.manual_seed(1)
x = torch.randn(6, 512, device="cuda").bfloat16()
w = torch.randn(1000, 512, device="cuda").bfloat16()
nw = torch.ones(512, device="cuda").bfloat16()
ids, u = torch.randint(0, 1000, (2, 2), dtype=torch.int32, device="cuda"), torch.rand(2, 3, device="cuda")
codes, scales = torch.empty(6, 512, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(6, device="cuda")
ws = q4t.VerifyDrafts(2, 2, 1000)
def step():
    q4t.residual_rmsnorm_fp8(x, None, nw, codes, scales)
    wc, wsc = q4t.quantize_rows_fp8(w)
    logits = q4t.linear(codes, wc, x_scale=scales, w_scale=wsc)
    return logits, ws(logits, ids, u)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    logits, out = step()
graph.replay()
torch.cuda.synchronize()
want_logits, want = step()
assert torch.equal(logits, want_logits)
assert all(torch.equal(out[k], want[k]) for k in want)
q4t.linear_status()
print("captured")
"""


def test_first_calls_of_a_process_inside_a_capture(q4t, gpu_lib):
    """No operator needs a call outside a graph first."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL % root], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_refused_steps_change_nothing(q4t, gpu_lib):
    """What a verification refuses is refused before the stack or the residual addition have changed x."""
    dl = q4t.DeviceLayer.from_host(synth.make_layer(E=8, hs=256, moe_is=128, shared_is=128, seed=1))
    nw, w = head_weights(100, 256, 5)
    stack, head = q4t.DecodeStack([dl], 6, 2), q4t.VerifyHead(nw, w, 2, 2)
    x = torch.randn(6, 256, device="cuda").bfloat16()
    before = x.clone()
    ids, u = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, device="cuda")
    for bad in (dict(draft_ids=ids.long()), dict(draft_ids=ids[:, :1]), dict(draft_ids=None), dict(uniforms=u.double()), dict(uniforms=u.cpu()),
                dict(uniforms=u.t()), dict(temperature=torch.ones(3, device="cuda")), dict(draft_len=torch.ones(2, device="cuda")),
                dict(draft_logits=torch.zeros(4, 99, device="cuda")), dict(draft_logits=torch.zeros(4, 100, device="cuda")),
                dict(draft_logits=torch.zeros(100, 4, device="cuda").bfloat16().t())):
        args = dict(dict(draft_ids=ids, uniforms=u), **bad)
        with pytest.raises(q4t.Q4TError):
            stack.verify(x, head, **args)
        with pytest.raises(q4t.Q4TError):
            head(x, y=x.clone(), **args)
    assert torch.equal(x, before)


def test_a_head_that_does_not_fit_is_refused_before_x_changes(q4t, gpu_lib):
    dl = q4t.DeviceLayer.from_host(synth.make_layer(E=8, hs=256, moe_is=128, shared_is=128, seed=1))
    stack = q4t.DecodeStack([dl], 6, 2)
    x = torch.randn(6, 256, device="cuda").bfloat16()
    before = x.clone()
    ids, u = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, device="cuda")
    nw, w = head_weights(100, 512, 5)
    with pytest.raises(q4t.Q4TError):
        stack.verify(x, q4t.VerifyHead(nw, w, 2, 2), ids, u)
    assert torch.equal(x, before)


def test_overlapping_draft_rows_are_refused_before_x_changes(q4t, gpu_lib):
    dl = q4t.DeviceLayer.from_host(synth.make_layer(E=8, hs=256, moe_is=128, shared_is=128, seed=1))
    nw, w = head_weights(100, 256, 5)
    stack, head = q4t.DecodeStack([dl], 6, 2), q4t.VerifyHead(nw, w, 2, 2)
    x = torch.randn(6, 256, device="cuda").bfloat16()
    before = x.clone()
    ids, u = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, device="cuda")
    one = torch.zeros(1, 100, device="cuda").bfloat16()
    for bad in (one.expand(4, 100), torch.zeros(200, device="cuda").bfloat16().as_strided((4, 100), (30, 1))):
        with pytest.raises(q4t.Q4TError):
            stack.verify(x, head, ids, u, draft_logits=bad)
        with pytest.raises(q4t.Q4TError):
            head(x, ids, u, y=x.clone(), draft_logits=bad)
    assert torch.equal(x, before)


@pytest.mark.parametrize("B,n,hs,V", [(1, 1, 256, 517), (4, 3, 512, 3001), (8, 3, 2048, 8192), (3, 7, 1040, 1000)])
def test_logits_of_the_e4m3_head(q4t, gpu_lib, B, n, hs, V):
    """The head's logits are the product of what its norm and its weight's layout left, in 64 bits: at most hs / 32 + 32 additions
    of an fp32 ulp of S each, four fp32 roundings, and one bf16 rounding.  Against the product of the unrounded operands the whole error is the two
    e4m3 roundings': each uniform within 2^-4 of a value at most, so 2^-4 / sqrt(3) in the root mean square, in quadrature, relative to the
    root of the summed squares; a quarter more covers the spread over a finite number of logits, the codes below 2^-6 and the bf16 rounding."""
    T = B * (n + 1)
    nw, w = head_weights(V, hs, V)
    head = q4t.VerifyHead(nw, w, B, n)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (2 * torch.randn(T, hs, generator=g, device="cuda")).bfloat16()
    head(x, torch.zeros(B, n, dtype=torch.int32, device="cuda"), torch.rand(B, n + 1, generator=g, device="cuda"))
    a, b = head.codes.float().double() * head.scales.double()[:, None], head.head.float().double() * head.head_scale.double()[:, None]
    want, S = a @ b.t(), a.abs() @ b.abs().t()
    tol = ((hs / 32 + 32) * 2.0 ** -23 + 4 * 2.0 ** -24) * S
    assert ((head.logits.double() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol)).all()
    v = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt() * nw.double()
    S2 = (v.square() @ w.double().square().t()).sqrt()
    assert float((head.logits.double() - v @ w.double().t()).norm() / S2.norm()) <= 1.25 * 2.0 ** 0.5 * 2.0 ** -4 / 3.0 ** 0.5
