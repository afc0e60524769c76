"""The serving operators at values, lengths and tables past those of test_gpu_serve.py, whose helpers and tolerances they use."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_serve import TYPES, do_verify, gen, ints, verify64  # noqa: E402

# ---- verification of drafts ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,first,second", [(3, 0, 1), (259, 17, 18), (8192, 40, 4099), (128256, 5, 100003)])
def test_verify_greedy_takes_the_first_of_two_zeros(dtype, V, first, second):
    # -0 and +0 are equal: whichever sign comes first, the first of them is the first maximum
    u = torch.full((1, 2), 0.5, device="cuda")
    for a, b in ((-0.0, 0.0), (0.0, -0.0), (-0.0, -0.0)):
        target = torch.full((1, 2, V), -1.0, device="cuda")
        target[..., first], target[..., second] = a, b
        for drafted, want in ((first, [first, first]), (second, [first, -1])):
            got, n = do_verify(target.to(TYPES[dtype][0]), None, ints([[drafted]]), u, "logits", 0.0, None, dtype)
            assert got.tolist() == [want] and n[0] == 1 + (drafted == first)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T", [1e-6, 1e-5, 0.8, 3.0])
@pytest.mark.parametrize("offset,spread", [
    (2e4, 3.0), (-3e5, 3.0), (6e4, 3000.0), (-1e9, 1e3),  # a step of fp32 is more than a thousand halvings at the lowest temperatures
    (1e30, 0.0), ("lowest", 0.0), ("largest", 0.0)])      # all alike, as in a row that is masked as a whole: uniform
def test_verify_logits_far_from_zero(dtype, T, offset, spread):
    V, top = 1000, torch.finfo(TYPES[dtype][0]).max
    base = {"lowest": -top, "largest": top}.get(offset, offset)
    if abs(base) > top:
        pytest.skip("past the type's range")
    target = base + spread * torch.rand(1, 2, V, generator=gen(1), device="cuda", dtype=torch.float64)
    target = target.to(TYPES[dtype][0])
    target[0, :, 7], target[0, :, 8] = -float("inf"), float("nan")
    x, u = ints([[3]]), torch.tensor([[0.9, 0.6004]], device="cuda")  # 0.6004 of 997 or 998 equal weights is inside an entry
    for t, draft, xs, us in ((target, None, x, u), (target[:, :1].contiguous(), None, x, u[:, 1:].contiguous()),
                             (target, target[:, 1:].roll(1, -1).contiguous(), x, u)):
        if spread == 0 and draft is not None:
            continue  # p - q of equal rows is a matter of rounding
        got, n = do_verify(t, draft, xs, us, "logits", T, None, dtype)
        # the record's 1e-6 is the fp32 number, which is not below itself: the oracle, which compares it in 64 bits, gets the next one
        # (weights of so low a temperature are one or zero with either)
        want, m = verify64(t, draft, xs, us, "logits", float(np.nextafter(np.float32(T), np.float32(1))) if T == 1e-6 else T)
        assert np.array_equal(n, m) and np.array_equal(got, want)
