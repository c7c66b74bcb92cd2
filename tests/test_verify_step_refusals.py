"""Refusals of the verify step's operators that precede any device work (no GPU needed)."""
import ctypes as C

import pytest
import torch

P = C.c_void_p(4096)     # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib(q4t):
    return q4t.load()


def refused(lib, rc, text):
    assert rc == -1, rc
    assert text in lib.q4t_last_error().decode()


def test_norm_fp8(lib):
    f = lib.q4t_residual_rmsnorm_fp8

    def call(x=P, y=P, x_out=P, w=P, codes=P, scales=P, h=None, T=2, hs=64, eps=1e-6):
        return f(x, y, x_out, w, 0.0, codes, scales, h, T, hs, eps, None)
    assert call(T=0) == 0 and call(T=-3) == 0
    for k in ("x", "codes", "scales"):
        refused(lib, call(**{k: None}), "null pointer")
    refused(lib, call(x_out=None), "destination")
    refused(lib, call(y=None), "nothing is added")
    for hs in (0, -8, 12, 32776):
        refused(lib, call(hs=hs), "multiple of 8")
    refused(lib, call(eps=-1.0), "eps")
    refused(lib, call(eps=float("nan")), "eps")
    refused(lib, call(h=P), "of its own")
    for k in ("x", "y", "x_out", "w", "h"):
        refused(lib, call(**{k: C.c_void_p(4104)}), "16-byte")
    refused(lib, call(codes=C.c_void_p(4100)), "8-byte")


def test_quantize_rows(lib):
    f = lib.q4t_quantize_rows_fp8
    assert f(P, P, P, 0, 64, None) == 0
    refused(lib, f(None, P, P, 2, 64, None), "null pointer")
    refused(lib, f(P, P, P, 2, 60, None), "multiple of 8")
    refused(lib, f(P, P, P, 2, 32776, None), "multiple of 8")
    refused(lib, f(C.c_void_p(4104), P, P, 2, 64, None), "16-byte")
    refused(lib, f(P, C.c_void_p(4097), P, 2, 64, None), "8-byte")


def test_python_arguments(q4t):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(q4t.Q4TError, match="CUDA tensor"):
        q4t.quantize_rows_fp8(x)
    with pytest.raises(q4t.Q4TError, match="not supported"):
        q4t.quantize_rows_fp8(x.float())
    with pytest.raises(q4t.Q4TError, match="two dimensions"):
        q4t.quantize_rows_fp8(x[0])
    with pytest.raises(q4t.Q4TError, match="two dimensions"):
        q4t.residual_rmsnorm_fp8(x[0], None, None, None, None)


def test_verify_drafts(lib, q4t):
    need = lib.q4t_verify_drafts_workspace_bytes(4, 3, 1000)
    assert need > 0
    for bad in ((0, 3, 1000), (4, 0, 1000), (4, 65, 1000), (4, 3, 0), (30000, 3, 1000)):
        assert lib.q4t_verify_drafts_workspace_bytes(*bad) == 0

    def call(ws=P, bytes_=1 << 30, **k):
        a = q4t.VerifyArgs(4096, None, 0, 0, 0, 4, 3, 1000, 4096, None, None, 4096, 4096, 4096, None)
        for name, v in k.items():
            setattr(a, name, v)
        return lib.q4t_verify_drafts(C.byref(a), ws, bytes_, None)
    assert lib.q4t_verify_drafts(None, P, need, None) == -1
    assert call(B=0) == 0 and call(B=-1) == 0
    refused(lib, call(n=0), "n out of range")
    refused(lib, call(n=65), "n out of range")
    refused(lib, call(V=0), "V out of range")
    refused(lib, call(V=(1 << 30) + 1), "V out of range")
    refused(lib, call(B=10000), "too many rows")
    for f in ("target_logits", "draft_ids", "uniforms", "tokens", "accepted"):
        refused(lib, call(**{f: None}), "null pointer")
    refused(lib, call(target_ld=999), "shorter than V")
    refused(lib, call(draft_logits=4096, draft_ld=10), "shorter than V")
    refused(lib, call(target_logits=4097), "aligned")
    refused(lib, call(target_logits=4098, logits_f32=1), "aligned")
    refused(lib, call(ws=C.c_void_p(4104)), "16-byte")
    assert call(bytes_=need - 1) == -2 and b"workspace" in lib.q4t_last_error()
    assert call(ws=None) == -2


def test_linear(lib, q4t):
    def call(**k):
        a = q4t.LinearArgs(4096, 4096, 4, 8, 64, 0, 0, 0, None, None, None, 0, 0, None, 0, 0, 8192)
        for name, v in k.items():
            setattr(a, name, v)
        return lib.q4t_linear(C.byref(a), None)
    assert lib.q4t_linear(None, None) == -1
    assert call(M=0) == 0 and call(M=-1) == 0
    refused(lib, call(N=0), "invalid GEMM dims")
    refused(lib, call(K=-4), "invalid GEMM dims")
    for f in ("x", "w", "out"):
        refused(lib, call(**{f: None}), "null pointer")
    refused(lib, call(activation=3), "activation")
    refused(lib, call(activation=-1), "activation")
    refused(lib, call(x_scale=4096), "e4m3")
    refused(lib, call(w_scale=4096), "e4m3")
    for f, v in (("ldx", 56), ("ldw", 63), ("ldo", 7), ("ldr", 7)):
        refused(lib, call(**{f: v}), "shorter than its row")
    refused(lib, call(x=4104), "16 bytes")
    refused(lib, call(w=4098), "16 bytes")
    refused(lib, call(ldx=68), "16 bytes")
    refused(lib, call(K=60), "16 bytes")
    refused(lib, call(fp8=1, ldw=72), "16 bytes")
    refused(lib, call(out=8193), "aligned to their types")
    refused(lib, call(out=8194, out_f32=1), "aligned to their types")
    refused(lib, call(bias=4097), "aligned to their types")
    refused(lib, call(residual=8192, ldr=16), "in place")
    refused(lib, call(residual=8192, out_f32=1), "in place")
    refused(lib, call(M=2 ** 31 - 1, N=2 ** 31 - 1, ldo=2 ** 31, ldr=2 ** 31), "too large")
    refused(lib, call(K=2 ** 30), "too large")


def test_python_linear_and_verify_arguments(q4t):
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    with pytest.raises(q4t.Q4TError, match="CUDA tensor"):
        q4t.linear(x, w)
    with pytest.raises(q4t.Q4TError, match="activation"):
        q4t.linear(x, w, activation="tanh")
    with pytest.raises(q4t.Q4TError, match="scales belong"):
        q4t.linear(x, w, x_scale=torch.ones(4))
    with pytest.raises(q4t.Q4TError, match="two dimensions"):
        q4t.linear(x[0], w)
    with pytest.raises(q4t.Q4TError, match="not supported"):
        q4t.linear(x.float(), w)
    with pytest.raises(q4t.Q4TError, match="out of range"):
        q4t.VerifyDrafts(2, 65, 100, device="cpu")


def test_outputs_over_operands_are_refused(lib, q4t):
    """Each output against each other buffer: the last byte that overlaps is refused.  (One that does not is covered by the calls
    on real buffers.)"""
    T, hs = 3, 64
    x, y, w, codes, scales, h, x_out = (4096 * (i + 1) for i in range(7))

    def norm(**k):
        a = dict(x=x, y=y, x_out=x_out, w=w, codes=codes, scales=scales, h=h)
        a.update(k)
        return lib.q4t_residual_rmsnorm_fp8(a["x"], a["y"], a["x_out"], a["w"], 0.0, a["codes"], a["scales"], a["h"], T, hs, 1e-6, None)
    for at in (x + 16, x - 16, y + T * hs * 2 - 16):
        refused(lib, norm(x_out=at), "x_out must be")
    refused(lib, norm(x_out=x, y=x + 16), "x_out must be")
    refused(lib, norm(x_out=w), "x_out overlaps weight")
    for name, at in (("x", x + T * hs * 2 - 8), ("y", y), ("x_out", x_out + 8), ("weight", w)):
        refused(lib, norm(codes=at), f"codes overlaps {name}")
    refused(lib, norm(scales=codes + T * hs - 4), "scales overlaps codes")
    refused(lib, norm(h=codes), "h overlaps codes")
    refused(lib, norm(h=x + 32), "h overlaps x")
    refused(lib, norm(scales=scales + 2), "4-byte")
    refused(lib, lib.q4t_quantize_rows_fp8(x, x + 8, scales, T, hs, None), "codes overlaps x")
    refused(lib, lib.q4t_quantize_rows_fp8(x, codes, codes, T, hs, None), "scales overlaps codes")
    refused(lib, lib.q4t_quantize_rows_fp8(x, codes, x + 4, T, hs, None), "scales overlaps x")
    refused(lib, lib.q4t_quantize_rows_fp8(x, codes, scales + 1, T, hs, None), "4-byte")

    base = 1 << 20

    def linear(**k):   # x [4, 64], w [8, 64], out [4, 8]
        a = q4t.LinearArgs(base, 2 * base, 4, 8, 64, 0, 0, 0, None, None, None, 0, 0, None, 0, 0, 3 * base)
        for name, v in k.items():
            setattr(a, name, v)
        return lib.q4t_linear(C.byref(a), None)
    refused(lib, linear(out=base + 4 * 128 - 2), "out overlaps x")
    refused(lib, linear(out=2 * base - 62), "out overlaps w")
    refused(lib, linear(bias=3 * base + 62), "out overlaps bias")
    refused(lib, linear(residual=3 * base + 2), "out overlaps residual")
    refused(lib, linear(residual=3 * base + 32, ldr=16), "out overlaps residual")       # another pitch
    refused(lib, linear(residual=3 * base + 14, ldr=24, ldo=24), "out overlaps residual")   # one pitch, one shared column
    refused(lib, linear(residual=3 * base - 34, ldr=24, ldo=24), "out overlaps residual")   # the column before, of the row above
    refused(lib, linear(fp8=1, x_scale=3 * base + 60), "out overlaps x_scale")
    refused(lib, linear(fp8=1, w_scale=3 * base - 28), "out overlaps w_scale")
    refused(lib, linear(fp8=1, w_scale=3 * base + 98), "aligned to their types")
    refused(lib, linear(ldo=1 << 62), "too large")

    need = lib.q4t_verify_drafts_workspace_bytes(4, 3, 1000)
    target, draft, ids, lens, temp, u, tokens, accepted, probs, ws = (base * (i + 1) for i in range(10))

    def verify(ws=ws, **k):
        a = q4t.VerifyArgs(target, draft, 0, 0, 0, 4, 3, 1000, ids, lens, temp, u, tokens, accepted, probs)
        for name, v in k.items():
            setattr(a, name, v)
        return lib.q4t_verify_drafts(C.byref(a), C.c_void_p(ws), need, None)
    inputs = dict(target_logits=target + 16 * 2000 - 4, draft_logits=draft, draft_ids=ids + 44, draft_len=lens + 12,
                  temperature=temp, uniforms=u + 60)
    for name, at in inputs.items():
        for out in ("tokens", "accepted", "probs"):
            refused(lib, verify(**{out: at}), f"{out} overlaps {name}")
        refused(lib, verify(ws=at & -16), f"workspace overlaps {name}")
    refused(lib, verify(accepted=tokens + 60), "accepted overlaps tokens")
    refused(lib, verify(probs=accepted - 60), "probs overlaps accepted")
    refused(lib, verify(ws=probs), "workspace overlaps probs")
    for name in ("draft_ids", "draft_len", "temperature", "uniforms", "tokens", "accepted", "probs"):
        refused(lib, verify(**{name: 4097 * 2}), "4-byte")
    refused(lib, verify(target_ld=1 << 60), "too large")
    assert lib.q4t_verify_drafts_workspace_bytes(4, 3, (1 << 30) + 1) == 0


def test_verify_head_shape(q4t):
    for shape, fp8 in (((32, 24), True), ((32, 12), False), ((32,), True)):
        with pytest.raises(q4t.Q4TError, match="head_weight"):
            q4t.VerifyHead(None, torch.zeros(shape, dtype=torch.bfloat16), 1, 1, fp8=fp8)


@pytest.fixture
def step(q4t, monkeypatch):
    """A stack and a head that fits it, on the host; the list grows when the stack runs."""
    ran = []
    monkeypatch.setattr(q4t.DecodeStack, "__call__", lambda self, x, stream=None: ran.append(x))
    stack = object.__new__(q4t.DecodeStack)
    stack.layers, stack.T, stack.h = [type("Layer", (), {"hs": 256})()], 6, torch.empty(6, 256, dtype=torch.bfloat16)
    return stack, q4t.VerifyHead(None, torch.zeros(100, 256, dtype=torch.bfloat16), 2, 2, fp8=False), ran


IDS, U = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 3)


@pytest.mark.parametrize("x,text", [(torch.zeros(5, 256, dtype=torch.bfloat16), "contiguous"),           # too few rows
                                    (torch.zeros(7, 256, dtype=torch.bfloat16), "contiguous"),
                                    (torch.zeros(6, 128, dtype=torch.bfloat16), "contiguous"),
                                    (torch.zeros(6 * 256, dtype=torch.bfloat16), "contiguous"),
                                    (torch.zeros(6, 512, dtype=torch.bfloat16)[:, ::2], "contiguous"),   # strided
                                    (torch.zeros(6, 320, dtype=torch.bfloat16)[:, :256], "contiguous"),
                                    (torch.zeros(6, 256), "contiguous"),                                # another type
                                    (torch.zeros(6, 256, dtype=torch.float16), "contiguous"),
                                    (None, "contiguous"),
                                    (torch.zeros(6, 256, dtype=torch.bfloat16), "CUDA tensor")])
def test_rows_that_the_stack_would_read_past_are_refused(q4t, step, x, text):
    stack, head, ran = step
    with pytest.raises(q4t.Q4TError, match=text):
        stack.verify(x, head, IDS, U)
    assert not ran


def test_a_head_of_other_rows_is_refused_before_the_stack_runs(q4t, step):
    stack, head, ran = step
    other = q4t.VerifyHead(None, torch.zeros(100, 512, dtype=torch.bfloat16), 2, 2, fp8=False)
    with pytest.raises(q4t.Q4TError, match="the head takes rows of 512"):
        stack.verify(torch.zeros(6, 256, dtype=torch.bfloat16), other, IDS, U)
    assert not ran


def test_weights_that_no_step_could_use_are_refused_with_the_head(q4t):
    def head(norm=None, w=torch.zeros(100, 256, dtype=torch.bfloat16), eps=1e-6, fp8=False):
        return q4t.VerifyHead(norm, w, 2, 2, eps=eps, fp8=fp8)
    good = torch.zeros(256, dtype=torch.bfloat16)
    assert head(good).T == 6 and head().T == 6
    assert head(w=torch.zeros(100, 272, dtype=torch.bfloat16)[:, :256]).T == 6      # rows further apart
    for bad in (good.float(), good[:128], torch.zeros(512, dtype=torch.bfloat16)[::2], good.view(1, 256), 1.0,
                torch.zeros(264, dtype=torch.bfloat16)[4:260]):
        with pytest.raises(q4t.Q4TError, match="norm_weight"):
            head(bad)
    wide = torch.zeros(100, 264, dtype=torch.bfloat16)
    for bad in (torch.zeros(100, 256), torch.zeros(2, 32776, dtype=torch.bfloat16), torch.zeros(256, 100, dtype=torch.bfloat16).t(),
                wide[:, 4:260], torch.zeros(100, 260, dtype=torch.bfloat16)[:, :256], good.expand(100, 256)):
        with pytest.raises(q4t.Q4TError, match="head_weight"):
            head(w=bad)
    for eps in (-1e-6, float("nan")):
        with pytest.raises(q4t.Q4TError, match="eps"):
            head(eps=eps)


def test_draft_rows_that_overlap_are_refused_by_the_check(q4t):
    v = q4t.VerifyDrafts(2, 2, 100, device="cpu")
    bf16 = torch.bfloat16
    v.check(IDS, U)
    for good in (torch.zeros(4, 100, dtype=bf16), torch.zeros(4, 107, dtype=bf16)[:, :100], torch.zeros(4, 101, dtype=bf16)[:, 1:]):
        v.check(IDS, U, good)
    for bad in (torch.zeros(1, 100, dtype=bf16).expand(4, 100), torch.zeros(400, dtype=bf16).as_strided((4, 100), (99, 1))):
        with pytest.raises(q4t.Q4TError, match="rows overlap"):
            v.check(IDS, U, bad)
    one = q4t.VerifyDrafts(1, 1, 100, device="cpu")      # the stride of a single row does not matter
    one.check(IDS[:1, :1], U[:1, :2], torch.zeros(100, dtype=bf16).as_strided((1, 100), (0, 1)))


def test_draft_logits_in_the_logits_of_the_step_are_refused(q4t, step):
    """They would be overwritten before they are read."""
    stack, head, ran = step
    for bad in (head.logits[:4], head.logits[2:]):
        with pytest.raises(q4t.Q4TError, match="head's own logits"):
            stack.verify(torch.zeros(6, 256, dtype=torch.bfloat16), head, IDS, U, draft_logits=bad)
        with pytest.raises(q4t.Q4TError, match="head's own logits"):
            head(torch.zeros(6, 256, dtype=torch.bfloat16), IDS, U, draft_logits=bad)
    assert not ran


def test_checks_alone(lib, q4t):
    """The checks refuse what the calls refuse, without a GPU; what they accept they only look at."""
    base = 1 << 20
    good = q4t.LinearArgs(base, 2 * base, 4, 8, 64, 0, 0, 0, None, None, None, 0, 0, None, 0, 0, 3 * base)
    assert lib.q4t_linear_check(C.byref(good)) == 0
    refused(lib, lib.q4t_linear_check(None), "null")
    good.out = base + 2
    refused(lib, lib.q4t_linear_check(C.byref(good)), "out overlaps x")
    good.M = 0
    assert lib.q4t_linear_check(C.byref(good)) == 0
    need = lib.q4t_verify_drafts_workspace_bytes(4, 3, 1000)
    v = q4t.VerifyArgs(base, None, 0, 0, 0, 4, 3, 1000, 2 * base, None, None, 3 * base, 4 * base, 5 * base, None)
    assert lib.q4t_verify_drafts_check(C.byref(v), 6 * base, need) == 0
    assert lib.q4t_verify_drafts_check(C.byref(v), 6 * base, need - 1) == -2
    refused(lib, lib.q4t_verify_drafts_check(None, 6 * base, need), "null")
    v.accepted = 4 * base + 60
    refused(lib, lib.q4t_verify_drafts_check(C.byref(v), 6 * base, need), "accepted overlaps tokens")
    v.B = 0
    assert lib.q4t_verify_drafts_check(C.byref(v), 6 * base, need) == 0
