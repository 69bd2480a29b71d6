"""Routing, the gradient for stored values and distillation where they can go wrong: large masks, near choices, crowded columns, waits that run
out.  Against the definitions in 64 bits and the tolerances of test_gpu_scores."""
import pytest
import torch

from csrspmm_b200 import ops
from test_gpu_scores import _gen, check_distill, teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("t", [0.5, 1.0, 2.0, 3.0])
@pytest.mark.parametrize("V", [300, 20000, 150_000, 600_000])
def test_distill_of_rows_masked_by_large_numbers(cuda_lib, V, t, dtype):
    """Masks that are finite: whole rows of them (a uniform distribution), rows with a few columns left, and rows whose columns are left only
    where they begin, so that threads, warps and whole parts of a row see nothing but the mask."""
    masks = [-1e10, -1e20, -1e30, torch.finfo(dtype).min]
    T = 3 * len(masks)
    x = torch.randn(T, V, device="cuda", generator=_gen(V)).to(dtype)
    rp, ci, va = teacher(T, V, [6] * T, 3)
    hit = ci.long().view(T, 6)
    hit[2::3] = torch.arange(6, device="cuda") * 5
    ci = hit.flatten().int()
    for i, mask in enumerate(masks):
        taught = x[3 * i + 1, hit[3 * i + 1]]
        x[3 * i : 3 * i + 2] = mask
        x[3 * i + 1, hit[3 * i + 1]] = taught
        x[3 * i + 2, 40:] = mask
    check_distill(x, rp, ci, va, t)


@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("V", [300, 20000, 150_000, 600_000])
def test_distill_of_rows_about_where_the_exponent_is_taken_another_way(cuda_lib, V, sign):
    """Maxima on both sides of |m log2(e)| = 2^24 among the threads, warps and parts of a row: whole numbers next to 2^24 ln(2) = 11629080."""
    x = torch.randint(-9, 10, (4, V), device="cuda", generator=_gen(V)).float()
    x[:, : V // 3] -= 12.0
    x[1, V // 2 :] -= 7.0
    check_distill(x + sign * 11629080.0, *teacher(4, V, [6] * 4, 5))


def test_the_gradients_of_a_matrix_of_nearly_2_to_31_rows(cuda_lib):
    M, Kd = 2 ** 31 - 2, 5
    rp = torch.zeros(M + 1, dtype=torch.int32, device="cuda")
    rp[M - 2] = 2  # two entries in row M - 3, none in M - 2, one in M - 1
    rp[M - 1] = 2
    rp[M] = 3
    ci = torch.tensor([4, 0, 4], dtype=torch.int32, device="cuda")
    va = torch.tensor([2.0, 3.0, 5.0], device="cuda")
    G, B = torch.zeros(M, 1, device="cuda"), torch.tensor([[1.0], [0.0], [0.0], [0.0], [7.0]], device="cuda")
    G[M - 3], G[M - 1] = 11.0, 13.0
    assert ops.sddmm(rp, ci, G, B).tolist() == [77.0, 11.0, 91.0]
    assert torch.ops.csrspmm_b200.spmm_transposed(rp, ci, va, G, Kd, 1.0).flatten().tolist() == [33.0, 0.0, 0.0, 0.0, 87.0]
