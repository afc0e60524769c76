"""The serving operators at values, lengths and tables past those of test_gpu_serve.py, whose helpers and tolerances they use."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_serve import TYPES, do_verify, ints  # noqa: E402

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
