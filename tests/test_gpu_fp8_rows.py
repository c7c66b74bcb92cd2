"""q4t_residual_rmsnorm_fp8 and q4t_quantize_rows_fp8 against the formulas in 64 bits.

Tolerances.  v is computed in fp32 from bf16 inputs: a sum of squares of at most 32 fused steps per thread and 10
additions of partial sums (each 2^-24 of the sum at most, halved by the square root), then a division, an addition, a
reciprocal root and two products: (42/2 + 6) * 2^-24 < 2^-19 relative.  The scale adds a division, the code's
argument a reciprocal and a product.  A code is off by half an e4m3 step: 2^-4 of the value, or 2^-10 where
the code is subnormal (step 2^-9); h by half a bf16 step, 2^-8 of the value."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu
REL = 2.0 ** -19
MIN_AMAX = 2.0 ** -64


def inputs(T, hs, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(T, hs, generator=g, device="cuda") * spread).bfloat16()
    y = torch.randn(T, hs, generator=g, device="cuda").bfloat16()
    w = (torch.randn(hs, generator=g, device="cuda") * 0.2 + 1.0).bfloat16()
    return x, y, w


def outputs(T, hs):
    return (torch.full((T, hs), 0x55, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
            torch.full((T,), -1.0, device="cuda"))


def formula(x, y, w, offset, eps):
    r = x if y is None else (x.float() + y.float()).bfloat16()
    v = r.double()
    v = v / (v.square().mean(dim=1, keepdim=True) + eps).sqrt()
    if w is not None:
        v = v * (w.double() + offset)
    return r, v


def check_rows(codes, scales, v):
    want = v.abs().amax(dim=1).clamp_min(MIN_AMAX) / 448.0
    assert ((scales.double() - want).abs() <= 2 * REL * want).all()
    t = v / want[:, None]
    off = (codes.float().double() - t).abs()
    assert (off <= torch.maximum(t.abs() * 2.0 ** -4, torch.full_like(t, 2.0 ** -10)) + 4 * REL * t.abs()).all()


@pytest.mark.parametrize("T,hs", [(1, 8), (1, 2048), (3, 24), (5, 1000), (130, 2560), (2, 8192), (3, 32768), (4097, 264)])
@pytest.mark.parametrize("with_y,with_w,offset,with_h", [(True, True, 0.0, False), (True, True, 1.0, True),
                                                        (False, True, 0.0, True), (True, False, 0.0, False),
                                                        (False, False, 0.0, False)])
def test_norm_against_the_formula(q4t, gpu_lib, T, hs, with_y, with_w, offset, with_h):
    x, y, w = inputs(T, hs, T * 7 + hs, spread=3.0)
    y, w = y if with_y else None, w if with_w else None
    codes, scales = outputs(T, hs)
    x_out = torch.empty_like(x) if with_y else None
    h = torch.empty_like(x) if with_h else None
    before = x.clone()
    q4t.residual_rmsnorm_fp8(x, y, w, codes, scales, x_out=x_out, h=h, eps=1e-6, weight_offset=offset)
    r, v = formula(x, y, w, offset, 1e-6)
    assert torch.equal(x, before)
    if with_y:
        assert torch.equal(x_out, r)
    if with_h:
        assert ((h.double() - v).abs() <= v.abs() * (2.0 ** -8 + 2 * REL)).all()
    check_rows(codes, scales, v)


@pytest.mark.parametrize("into", ["x", "y"])
def test_norm_in_place(q4t, gpu_lib, into):
    x, y, w = inputs(37, 2048, 5)
    r, v = formula(x, y, w, 0.0, 1e-5)
    codes, scales = outputs(37, 2048)
    out = x if into == "x" else y
    q4t.residual_rmsnorm_fp8(x, y, w, codes, scales, x_out=out, eps=1e-5)
    assert torch.equal(out, r)
    check_rows(codes, scales, v)


@pytest.mark.parametrize("rows,K", [(1, 8), (97, 2560), (2, 32768), (1000, 72), (5, 8200)])
def test_quantize_rows(q4t, gpu_lib, rows, K):
    x, _, _ = inputs(rows, K, rows + K, spread=0.02)
    codes, scales = q4t.quantize_rows_fp8(x)
    check_rows(codes, scales, x.double())
    # the largest element of a row is its 448
    assert (codes.float().abs().amax(dim=1) == 448.0).all()


def test_rows_at_the_ends_of_the_range(q4t, gpu_lib):
    """Zero rows, one element, the type's largest and smallest values, NaN and infinity."""
    big, tiny = torch.finfo(torch.bfloat16).max, 2.0 ** -126
    x = torch.zeros(8, 64, device="cuda")
    x[1, 5] = -3.0
    x[2] = big
    x[3] = tiny
    x[4, 7] = float("nan")
    x[5, 9] = float("inf")
    x[6, 63] = float("-inf")
    x[7] = torch.linspace(-1, 1, 64, device="cuda")
    x = x.bfloat16()
    codes, scales = q4t.quantize_rows_fp8(x)
    fine = [0, 1, 2, 3, 7]
    check_rows(codes[fine], scales[fine], x[fine].double())
    assert (codes[0].view(torch.uint8) & 0x7f == 0).all()
    assert scales[4:7].isnan().all() and codes[4:7].float().isnan().all()
    # the same through the norm: row 2's sum of squares leaves fp32
    codes, scales = outputs(8, 64)
    q4t.residual_rmsnorm_fp8(x, None, None, codes, scales, eps=1e-6)
    fine = [0, 1, 3, 7]
    check_rows(codes[fine], scales[fine], formula(x[fine], None, None, 0.0, 1e-6)[1])
    bad = [2, 4, 5, 6]
    assert scales[bad].isnan().all() and codes[bad].float().isnan().all()


def test_a_bad_row_leaves_the_others_alone(q4t, gpu_lib):
    x, y, w = inputs(9, 512, 3)
    want, swant = outputs(9, 512)
    q4t.residual_rmsnorm_fp8(x, y, w, want, swant, x_out=torch.empty_like(x))
    y[4, 100] = float("nan")
    got, sgot = outputs(9, 512)
    q4t.residual_rmsnorm_fp8(x, y, w, got, sgot, x_out=torch.empty_like(x))
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.equal(got.view(torch.uint8)[keep], want.view(torch.uint8)[keep]) and torch.equal(sgot[keep], swant[keep])
    assert sgot[4].isnan()


def test_rows_behind_the_last_stay(q4t, gpu_lib):
    x, _, _ = inputs(6, 256, 1)
    codes, scales = outputs(6, 256)
    gpu_lib.q4t_quantize_rows_fp8(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), 4, 256, None)
    torch.cuda.synchronize()
    assert (codes[4:].view(torch.uint8) == 0x55).all() and (scales[4:] == -1).all()


def test_on_another_stream_and_in_a_graph(q4t, gpu_lib):
    x, y, w = inputs(33, 2048, 11)
    want, swant = outputs(33, 2048)
    q4t.residual_rmsnorm_fp8(x, y, w, want, swant, x_out=torch.empty_like(x))
    codes, scales = outputs(33, 2048)
    out = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    q4t.residual_rmsnorm_fp8(x, y, w, codes, scales, x_out=out, stream=s)
    s.synchronize()
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, swant)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q4t.residual_rmsnorm_fp8(x, y, w, codes, scales, x_out=out)
    x.mul_(2)
    graph.replay()
    q4t.residual_rmsnorm_fp8(x, y, w, want, swant, x_out=torch.empty_like(x))
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, swant)


def division(v):
    """scale and e4m3(v / scale) of fp32 rows, with the divisions' own roundings (tensor by tensor: by a Python number a GPU tensor is
    multiplied with the number's reciprocal)."""
    top = v.abs().amax(dim=1).clamp_min(MIN_AMAX)
    scale = top / torch.full_like(top, 448.0)
    return (v / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def bf16_rows(rows, K, seed):
    """Values of many magnitudes; few-bit ones among them, whose quotients lie on rounding borders."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, K, generator=g, device="cuda") * torch.exp2(torch.randint(-60, 60, (rows, 1), generator=g, device="cuda").float())
    few = torch.randint(0, 32, (rows, K), generator=g, device="cuda").float() * torch.exp2(torch.randint(-8, 4, (rows, K), generator=g, device="cuda").float())
    x[::3] = (few * torch.where(torch.rand(rows, K, generator=g, device="cuda") < 0.5, -1.0, 1.0))[::3]
    x[1] = 0.0
    x[2, ::2] = -0.0
    return x.bfloat16()


@pytest.mark.parametrize("rows,K", [(96, 2560), (1201, 248), (1030, 504), (1100, 1016), (2050, 2048), (7, 8200), (3, 32768)])
def test_codes_are_the_division(q4t, gpu_lib, rows, K):
    """code = e4m3(v / scale) and scale = max / 448 bit for bit (v / scale rounded to fp32 first), signs of zeros included."""
    x = bf16_rows(rows, K, rows + K)
    codes, scales = q4t.quantize_rows_fp8(x)
    want, swant = division(x.float())
    assert torch.equal(scales, swant)
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("T,hs", [(3, 2048), (1030, 248), (1100, 512), (1050, 2560), (5, 16384), (2, 32768)])
def test_codes_of_a_norm_are_the_division(q4t, gpu_lib, T, hs):
    """Rows of ones of either sign have an rms of exactly one: v is the weight."""
    g = torch.Generator(device="cuda").manual_seed(T)
    sign = torch.where(torch.rand(T, hs, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    for i in range(3):
        w = bf16_rows(3, hs, hs + i)[i if i != 1 else 2]
        codes, scales = outputs(T, hs)
        q4t.residual_rmsnorm_fp8(sign.bfloat16(), None, w, codes, scales, eps=0.0)
        want, swant = division(sign * (w.float() + 0.0))   # the offset of zero takes the weight's -0 away
        assert torch.equal(scales, swant)
        assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))


def behind(rows, width, dtype, fill):
    return torch.full((rows + 3, width), fill, dtype=dtype, device="cuda")


@pytest.mark.parametrize("T,hs", [(1025, 8), (1033, 256), (1030, 264), (1029, 512), (1025, 520), (1030, 2560), (1027, 8192), (3, 8200), (1026, 8200),
                                  (2, 16384), (1025, 16392), (16385, 72)])
@pytest.mark.parametrize("with_y,with_w,offset,with_h", [(True, True, 1.0, True), (False, False, 0.0, False)])
def test_norm_of_many_and_of_long_rows(q4t, gpu_lib, T, hs, with_y, with_w, offset, with_h):
    """The forms that row counts above 1024 and row lengths choose; rows behind the last stay as they were."""
    x, y, w = inputs(T, hs, T + hs, spread=3.0)
    y, w = y if with_y else None, w if with_w else None
    codes, scales = behind(T, hs, torch.uint8, 0x55), behind(T, 1, torch.float32, -1.0)
    x_out = behind(T, hs, torch.bfloat16, 5.0) if with_y else None
    h = behind(T, hs, torch.bfloat16, 6.0) if with_h else None
    q4t.residual_rmsnorm_fp8(x, y, w, codes[:T].view(torch.float8_e4m3fn), scales[:T, 0], x_out=None if x_out is None else x_out[:T],
                             h=None if h is None else h[:T], eps=1e-6, weight_offset=offset)
    r, v = formula(x, y, w, offset, 1e-6)
    if with_y:
        assert torch.equal(x_out[:T], r) and (x_out[T:] == 5).all()
    if with_h:
        assert ((h[:T].double() - v).abs() <= v.abs() * (2.0 ** -8 + 2 * REL)).all() and (h[T:] == 6).all()
    check_rows(codes[:T].view(torch.float8_e4m3fn), scales[:T, 0], v)
    assert (codes[T:] == 0x55).all() and (scales[T:] == -1).all()


@pytest.mark.parametrize("rows,K", [(1027, 72), (1025, 256), (1031, 504), (1029, 1016), (1026, 1032), (1026, 2048), (1025, 16384), (1025, 16392), (9, 8200)])
def test_quantiser_of_many_and_of_long_rows(q4t, gpu_lib, rows, K):
    x, _, _ = inputs(rows, K, rows + K, spread=0.02)
    codes, scales = behind(rows, K, torch.uint8, 0x55), behind(rows, 1, torch.float32, -1.0)
    q4t.quantize_rows_fp8(x, codes[:rows].view(torch.float8_e4m3fn), scales[:rows, 0])
    check_rows(codes[:rows].view(torch.float8_e4m3fn), scales[:rows, 0], x.double())
    assert (codes[rows:] == 0x55).all() and (scales[rows:] == -1).all()
