"""q4t_verify_drafts against the definition in 64 bits (tests/verify_oracle.py).

Tokens and counts are compared exactly.  An acceptance is decided from fp32 exponentials: each is off by 2^-22 at most in
the exponential function, a rounding of its argument (at most 2^-24 of |z|, and e^z |z| <= 1) and 2^-24
per addition of at most 10 of them, so p and q are off by less than 16 * 2^-24 = 2^-20 each; draws
are 64-bit sums of at most V weights.  The seeds below leave every acceptance 2^-18 and every draw 1e-12 away from its
border, which each test asserts of its inputs before it looks at the outputs.  Probabilities: 2^-20 relative
and the fp32 they are stored in."""
import numpy as np
import pytest
import torch

from verify_oracle import verify

pytestmark = pytest.mark.gpu
PREL = 2.0 ** -19


def make(B, n, V, seed, draft=True, f32=False, ragged=False, greedy=0, ld=None):
    g = torch.Generator().manual_seed(seed)
    dt = torch.float32 if f32 else torch.bfloat16
    body = 2.0 * torch.randn(B, n + 1, V, generator=g)
    for r in body.view(-1, V):
        k = min(V, 12)
        r[torch.randperm(V, generator=g)[:k]] += 5.0 + 2.0 * torch.randn(k, generator=g)
    guess = body[:, :n] + 0.7 * torch.randn(B, n, V, generator=g)
    T = 0.6 + 0.6 * torch.rand(B, generator=g)
    T[:greedy] = 0.0
    s = {"target": body.to(dt), "draft": guess.to(dt) if draft else None, "T": T, "u": torch.rand(B, n + 1, generator=g),
         "lens": torch.randint(0, n + 1, (B,), generator=g, dtype=torch.int32) if ragged else None}
    if draft:
        q = torch.softmax(s["draft"].float() / T.clamp_min(0.3)[:, None, None], 2)
        s["ids"] = torch.multinomial(q.view(B * n, V), 1, generator=g).view(B, n).int()
    else:
        s["ids"] = guess.argmax(2).int()
    return s


def rows(t, ld=None):
    """[B, r, V] on the host -> [B*r, V] on the device, rows ld apart."""
    if t is None:
        return None
    flat = t.reshape(-1, t.shape[2])
    if ld is None:
        return flat.cuda()
    out = torch.full((flat.shape[0], ld), float("nan"), dtype=t.dtype, device="cuda")
    out[:, :t.shape[2]] = flat.cuda()
    return out[:, :t.shape[2]]


def run(q4t, s, ld=None, verifier=None, stream=None):
    B, n1, V = s["target"].shape
    v = verifier or q4t.VerifyDrafts(B, n1 - 1, V)
    c = lambda t: None if t is None else t.cuda()
    return v(rows(s["target"], ld), c(s["ids"]), c(s["u"]), draft_logits=rows(s["draft"], ld), temperature=c(s["T"]),
             draft_len=c(s["lens"]), stream=stream)


def expect(s):
    f = lambda t: None if t is None else t.float().numpy()
    tokens, accepted, probs, accept_margin, draw_margin = verify(
        f(s["target"]), s["ids"].numpy(), s["u"].numpy(), f(s["draft"]), None if s["T"] is None else s["T"].numpy(), None if s["lens"] is None else s["lens"].numpy())
    assert accept_margin > 2.0 ** -18 and draw_margin > 1e-12, "pick another seed: a decision of the inputs lies on its border"
    return tokens, accepted, probs


def compare(got, want):
    tokens, accepted, probs = want
    assert np.array_equal(got["accepted"].cpu().numpy(), accepted)
    assert np.array_equal(got["tokens"].cpu().numpy(), tokens)
    g = got["probs"].cpu().numpy().astype(np.float64)
    assert (np.abs(g - probs) <= PREL * probs + 1e-37).all()


@pytest.mark.parametrize("B,n,V", [(1, 1, 1), (1, 1, 2), (3, 2, 7), (2, 3, 1000), (5, 4, 4097), (4, 3, 32003), (2, 64, 333),
                                   (1, 2, 131072), (40, 1, 1025), (2, 2, 200001)])
@pytest.mark.parametrize("draft,f32", [(True, False), (False, False), (True, True), (False, True)])
def test_against_the_definition(q4t, gpu_lib, B, n, V, draft, f32):
    s = make(B, n, V, B * 1000 + n * 100 + V, draft, f32)
    compare(run(q4t, s), expect(s))


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("f32", [True, False])
def test_padded_batch_with_greedy_sequences_and_strided_rows(q4t, gpu_lib, draft, f32):
    s = make(9, 5, 5003, 42 + draft, draft, f32, ragged=True, greedy=3)
    s["lens"][4], s["lens"][5] = 0, 5
    want = expect(s)
    compare(run(q4t, s), want)
    for ld in (5008, 5021):
        compare(run(q4t, s, ld), want)
    s["lens"][5], s["lens"][4] = 99, -7      # clamped
    compare(run(q4t, s), want)


def test_defaults_without_temperature_and_lengths(q4t, gpu_lib):
    s = make(4, 3, 999, 5)
    s["T"] = None
    compare(run(q4t, s), expect(s))


@pytest.mark.parametrize("draft", [True, False])
def test_masked_and_special_logits(q4t, gpu_lib, draft):
    """-inf, the type's lowest value, NaN and +inf in masked places; rows that leave nothing; ids out of range."""
    s = make(8, 3, 771, 17, draft)
    t, low = s["target"], torch.finfo(torch.bfloat16).min
    t[0, :, 100:] = float("-inf")
    t[1, :, :700] = low
    t[2, :, ::2] = float("nan")
    t[3, 1] = float("-inf")          # nothing left in front of draft 1
    t[4, 0] = float("nan")           # nothing left in front of draft 0
    t[5, 2, 33], t[5, 2, 44] = float("inf"), float("inf")
    t[6] = low                       # the lowest value everywhere: uniform
    s["ids"][7, 1], s["ids"][0, 2] = -1, 771
    if draft:
        s["draft"][2, :, ::2] = float("nan")
        s["draft"][1, 1] = float("-inf")
        s["draft"][3, 0, 5] = float("inf")
    for i in range(8):
        s["ids"][i, 0] = int(torch.nan_to_num(t[i, 0].float(), nan=-1e38, posinf=1e38, neginf=-1e38).argmax())
    s["u"][:, 0] *= 0.01
    compare(run(q4t, s), expect(s))


def test_empty_rows_of_a_greedy_sequence_and_ties(q4t, gpu_lib):
    s = make(3, 2, 517, 3, greedy=3)
    s["target"][0, 0] = float("-inf")
    s["target"][1, 0] = 1.0                      # ties go to the lowest index
    s["ids"][1, 0] = 0
    s["target"][1, 1, 200], s["target"][1, 1, 300] = 99.0, 99.0
    s["ids"][1, 1] = 300
    s["u"][:] = float("nan")                     # not read
    got, want = run(q4t, s), expect(s)
    compare(got, want)
    assert got["tokens"][0].tolist() == [-1, -1, -1] and got["tokens"][1].tolist() == [0, 200, -1]


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -0.5, float("nan")])
def test_uniforms_at_and_past_their_ends(q4t, gpu_lib, u):
    for draft in (True, False):
        s = make(3, 2, 1500, 8, draft)
        s["target"][:, :, 1400:] = float("-inf")   # the last tokens have no weight
        s["target"][:, :, :10] = float("-inf")
        s["u"][:, 2] = u
        got = run(q4t, s)
        f = lambda t: None if t is None else t.float().numpy()
        tokens, accepted, *_ = verify(f(s["target"]), s["ids"].numpy(), s["u"].numpy(), f(s["draft"]), s["T"].numpy())
        assert np.array_equal(got["accepted"].cpu().numpy(), accepted)
        a = accepted
        drawn = got["tokens"].cpu().numpy()[np.arange(3), a]
        assert ((drawn >= 10) & (drawn < 1400)).all()
        if u != 1.0 - 2.0 ** -24:                   # within a rounding of the last border
            assert np.array_equal(drawn, tokens[np.arange(3), a])
        s["u"][:, :2] = u
        got = run(q4t, s)
        tokens, accepted, *_ = verify(f(s["target"]), s["ids"].numpy(), s["u"].numpy(), f(s["draft"]), s["T"].numpy())
        assert np.array_equal(got["accepted"].cpu().numpy(), accepted)


@pytest.mark.parametrize("T", [1e-30, 1e-3, 50.0, 1e30, float("inf")])
def test_temperatures_at_the_ends(q4t, gpu_lib, T):
    s = make(3, 2, 640, 21, True, True)
    s["target"][0, :, 17] = float("-inf")
    s["draft"][0, :, 18] = float("-inf")
    s["T"][:] = T
    if T == float("inf"):                       # a temperature that leaves all kept tokens alike
        s["T"][:] = 1e35
    want = expect(s)
    s["T"][:] = T
    compare(run(q4t, s), want)


def test_identical_distributions_accept_everything(q4t, gpu_lib):
    s = make(16, 4, 3001, 9)
    s["draft"] = s["target"][:, :4].clone()
    s["ids"] = torch.multinomial(torch.softmax(s["draft"].float().view(64, 3001), 1), 1).view(16, 4).int()
    got = run(q4t, s)
    assert (got["accepted"] == 4).all()
    # a refusal forced by the uniform leaves no difference: the draw is the target's own
    s["u"][:, 0] = 1.5
    compare(run(q4t, s), expect(s))


def test_outputs_follow_the_target(q4t, gpu_lib):
    """The first emitted token is distributed as the target says, whatever the drafter: 20000 sequences over 5
    tokens; the largest of 5 deviations stays under 5 standard deviations (probability of a false alarm < 3e-6)."""
    B = 20000
    tl = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.1])
    ql = torch.tensor([1.0, 0.5, -1.0, 0.7, 0.1])
    g = torch.Generator().manual_seed(0)
    ids = torch.multinomial(torch.softmax(ql, 0).expand(B, 5), 1, generator=g).int()
    u = torch.rand(B, 2, generator=g)
    v = q4t.VerifyDrafts(B, 1, 5)
    got = v(tl.expand(2 * B, 5).contiguous().cuda(), ids.cuda(), u.cuda(), draft_logits=ql.expand(B, 5).contiguous().cuda())
    first = got["tokens"][:, 0].cpu()
    p = torch.softmax(tl.double(), 0)
    share = torch.bincount(first.long(), minlength=5).double() / B
    assert ((share - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all()


def test_two_verifiers_on_two_streams_and_a_graph(q4t, gpu_lib):
    sa, sb = make(6, 3, 20011, 31), make(6, 3, 20011, 33)
    wa, wb = expect(sa), expect(sb)
    va, vb = q4t.VerifyDrafts(6, 3, 20011), q4t.VerifyDrafts(6, 3, 20011)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        ga = run(q4t, sa, verifier=va)
    with torch.cuda.stream(s2):
        gb = run(q4t, sb, verifier=vb)
    torch.cuda.synchronize()
    compare(ga, wa)
    compare(gb, wb)
    # captured once, replayed on other inputs in the same buffers
    t, ids, u = rows(sa["target"]), sa["ids"].cuda(), sa["u"].cuda()
    d, T = rows(sa["draft"]), sa["T"].cuda()
    va(t, ids, u, draft_logits=d, temperature=T)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = va(t, ids, u, draft_logits=d, temperature=T)
    for src, want in ((sb, wb), (sa, wa)):
        t.copy_(rows(src["target"])), d.copy_(rows(src["draft"]))
        ids.copy_(src["ids"]), u.copy_(src["u"]), T.copy_(src["T"])
        graph.replay()
        compare(out, want)
    a = run(q4t, sa, verifier=va)
    b = run(q4t, sa, verifier=va)
    assert all(torch.equal(a[k], b[k]) for k in a)


def long_rows(seed, draft):
    """Eight sequences of bf16 rows long enough for looked-up weights (more than 8192 tokens a CTA), each with values at an edge
    of what the table holds."""
    s = make(8, 2, 70001, seed, draft)
    g = torch.Generator().manual_seed(seed)
    pick = lambda k: torch.randperm(70001, generator=g)[:k]
    for t in [s["target"]] + ([s["draft"]] if draft else []):
        t[0, :, pick(30000)] = 0.0                                    # magnitudes below its smallest
        for v in (-0.0, 2.0 ** -12, -2.0 ** -13, 2.0 ** -20, -1e-39):
            t[0, :, pick(2000)] = v
        t[1, :, pick(50000)] = float("-inf")
        t[1, :, pick(9000)] = float("nan")
        t[1, :, pick(3000)] = torch.finfo(torch.bfloat16).min
        t[2] += 300.0                                                 # maxima that it does not serve
        t[3] -= 70.0
        t[4] -= 25.0
        t[7, :, pick(4000)] -= 110.0
        t[7, :, pick(300)] = -2040.0
        t[7, :, pick(300)] = -5000.0
        t[7, :, pick(300)] = -128.0
        t[7, :, pick(3)] = 127.5
    s["T"][5], s["T"][6], s["T"][7] = 0.15, 4.0, 0.9
    return s


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("refused", [True, False])
def test_long_rows_at_the_edges_of_the_weight_table(q4t, gpu_lib, draft, refused):
    s = long_rows(5 + draft, draft)
    s["u"][:, 0] = 1.5 if refused and draft else (0.999 if refused else 0.0)
    compare(run(q4t, s), expect(s))
    compare(run(q4t, s, 70013), expect(s))     # draft and target rows at different offsets in their 16 bytes


def test_least_weights_of_long_rows(q4t, gpu_lib):
    """A uniform of zero takes the first token that has any weight: one of e^-300 of the largest, none behind a mask."""
    s = make(2, 1, 70001, 3, False)
    s["target"][:, :, :5] = float("-inf")
    s["target"][:, :, 5] = float("nan")
    s["target"][:, :, 6] = -3000.0
    s["target"][0, :, 7], s["target"][1, :, 9] = -250.0, -250.0
    s["target"][1, :, 7:9] = torch.finfo(torch.bfloat16).min
    s["T"][:] = 0.9
    s["u"][:] = 0.0
    got = run(q4t, s)
    assert got["accepted"].tolist() == [1, 1] and got["tokens"][:, 1].tolist() == [7, 9]


def test_shifted_drafts_of_long_rows_leave_no_difference(q4t, gpu_lib):
    """softmax(l + 8) = softmax(l): a refusal that the uniform forces draws from the target's own distribution."""
    s = make(4, 2, 80000, 12)
    s["target"] = (s["target"].float().clamp(-16, 15) * 4).round().div(4).bfloat16()
    s["draft"] = (s["target"][:, :2].float() + 8).bfloat16()
    assert torch.equal(s["draft"].float(), s["target"][:, :2].float() + 8)
    s["u"][:, 0] = 1.5
    compare(run(q4t, s), expect(s))


def second_chunks(B, n, V, seed, draft, f32):
    """Rows of which a warp of the first kernel takes two chunks (512 fp32 or 1024 bf16 tokens), with what one chunk of a pair may hold."""
    L = 512 if f32 else 1024
    s = make(B, n, V, seed, draft, f32, ragged=True, greedy=6)
    parts = [s["target"]] + ([s["draft"]] if draft else [])
    for t in parts:
        t[0, :, 3 * L + 17] += 40.0                # maxima in the second chunk of a pair
        t[6, :, L + 5] += 40.0
        t[7, :, 5] += 30.0                          # a first chunk's maximum raised by the second's
        t[7, :, L + 9] += 33.0
        t[8, :, :L - 16] = float("-inf")            # the first, the second, both (and their neighbours)
        t[9, :, L - 16:2 * L + 16] = float("-inf")
        t[10, :, 2 * L - 16:4 * L + 16] = float("-inf")
        t[11, :, L + 3] = float("nan")
        t[12, :, 3 * L:4 * L] = float("nan")
        t[13, :, :L] = float("nan")
        t[1, :, 3 * L:3 * L + 40] = float("nan")    # greedy sequences
        t[2, :, :2 * L] = float("-inf")
        t[3, :, L + 200] = 60.0
        t[3, :, 3 * L + 200] = 60.0
        t[14] = torch.finfo(t.dtype).min
        t[15, :, :] = float("-inf")
        t[15, :, 2 * L + L // 2:2 * L + L // 2 + L] = 0.0
        t[16, :, V - 1] += 50.0
    s["target"][17, 0, L + 8] = float("inf")
    s["lens"][:18] = n
    return s


@pytest.mark.parametrize("B,n,V,draft,f32", [(64, 3, 16391, False, True), (32, 7, 20011, True, False), (40, 5, 8200, True, True), (64, 7, 12000, False, False)])
def test_second_chunks(q4t, gpu_lib, B, n, V, draft, f32):
    rows_ = B * (n + 1 + (n if draft else 0))
    per = 512 if f32 else 1024
    assert rows_ * ((V + 8 + per - 1) // per) // 2 >= 148 * 20     # the first kernel's rule for two chunks a warp
    s = second_chunks(B, n, V, V, draft, f32)
    want = expect(s)
    compare(run(q4t, s), want)
    compare(run(q4t, s, (V + 8) // 8 * 8 + 3), want)
    s["u"][:, 0] = 1.5                                             # every first draft refused
    compare(run(q4t, s), expect(s))


def nearly_equal(B, V, seed, f32):
    """Target and draft rows that agree to 1e-7, but for one unlikely token that the drafter favours and drafts.  fp32: noise of 2e-7 on every
    logit; bf16: one token in eight, of a total probability of 4e-8, has another logit."""
    g = torch.Generator().manual_seed(seed)
    dt = torch.float32 if f32 else torch.bfloat16
    t = (2.0 * torch.randn(B, 2, V, generator=g)).to(dt).float()
    x = torch.randint(0, V, (B, 1), generator=g)
    rare = torch.full((B, V), False)
    for b in range(B):
        rare[b, torch.randperm(V, generator=g)[:V // 8]] = True
    if f32:
        d = t[:, 0] + 2e-7 * torch.randn(B, V, generator=g)
    else:
        t[:, 0] = torch.where(rare, torch.full((B, V), -13.0), t[:, 0])
        d = t[:, 0] + torch.where(rare, torch.randint(-1, 2, (B, V), generator=g).float(), torch.zeros(B, V))
    t[:, 0].scatter_(1, x, -16.0)
    d.scatter_(1, x, -14.0)
    return {"target": t.to(dt), "draft": d[:, None].to(dt), "T": None, "u": torch.cat([torch.full((B, 1), 0.9), torch.rand(B, 1, generator=g)], 1),
            "lens": None, "ids": x.int()}


@pytest.mark.parametrize("B,V,seed,f32", [(24, 1001, 0, True), (24, 1001, 3, True), (12, 16000, 3, True), (12, 16000, 4, True), (2, 70001, 0, True),
                                              (2, 70001, 3, True), (24, 5001, 3, False), (12, 16000, 2, False), (12, 16000, 20, False), (2, 70001, 1, False)])
def test_draws_from_what_nearly_equal_distributions_leave(q4t, gpu_lib, B, V, seed, f32):
    """The weights are good to 1.5e-13 each, so a border of the draw to 3e-13 of the whole and, relative to the little that is left of it, to 3e-13 / left."""
    s = nearly_equal(B, V, seed, f32)
    p, q = (torch.softmax(s[k][:, 0].double(), 1) for k in ("target", "draft"))
    left = float((p - q).clamp_min(0).sum(1).min())
    assert 1e-8 < left < 1e-6
    tokens, accepted, probs, accept_margin, draw_margin = verify(
        s["target"].float().numpy(), s["ids"].numpy(), s["u"].numpy(), s["draft"].float().numpy())
    assert accept_margin > 2.0 ** -18 and draw_margin > 3e-13 / left and (accepted == 0).all()
    compare(run(q4t, s), (tokens, accepted, probs))
