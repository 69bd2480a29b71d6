"""Routing, the gradient for stored values and distillation where they can go wrong: large masks, near choices, crowded columns, waits that run
out.  Against the definitions in 64 bits and the tolerances of test_gpu_scores."""
import pytest
import torch

from csrspmm_b200 import ops
from test_gpu_scores import U, _gen, _rows, check_distill, route_f64, teacher

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("T,V", [(2, 6001), (2000, 6001), (12000, 3001), (3000, 30011), (8, 60_000), (300, 150_003), (4, 300_003)])
def test_distill_waits_that_run_out_leave_nan_and_nothing_unwritten(cuda_lib, monkeypatch, T, V, dtype):
    """Without a single attempt for a copy every row is given up: NaN in the loss and in every element of the gradient, but for rows without a
    teacher, which have nothing to wait for.  The context stays usable, and the next call is right."""
    lens = torch.full((T,), 5)
    lens[1::7] = 0
    rp, ci, va = teacher(T, V, lens, 6)
    x = torch.randn(T, V, device="cuda", generator=_gen(V)).to(dtype)
    taught = (lens > 0).cuda()
    good = ops.distill_loss_grad(x, rp, ci, va)
    monkeypatch.setenv("CSRSPMM_TEST_WAIT_LIMIT", "0")
    leaf = x.clone().requires_grad_(True)
    alone = ops.distill_loss(leaf, rp, ci, va)
    alone.sum().backward()
    out = torch.full((T, V), 7.0, device="cuda", dtype=dtype)  # memory that the gradient may get, with something in it
    del out
    loss, dx = ops.distill_loss_grad(x, rp, ci, va)
    torch.cuda.synchronize()
    for l, d in ((loss, dx), (alone.detach(), leaf.grad)):
        assert l[taught].isnan().all() and (l[~taught] == 0).all()
        assert d[taught].isnan().all() and (d[~taught] == 0).all()
    monkeypatch.delenv("CSRSPMM_TEST_WAIT_LIMIT")
    again = ops.distill_loss_grad(x, rp, ci, va)
    assert torch.equal(again[0], good[0]) and torch.equal(again[1], good[1]) and good[1].isfinite().all()


@pytest.mark.parametrize("twice", [False, True])
@pytest.mark.parametrize("T,V,n", [(3000, 30_011, 20_000), (3000, 30_011, 1000), (12_000, 3001, 3000), (12_000, 6001, 400), (80, 150_003, 40_000)])
def test_distill_of_one_long_row_among_short_ones(cuda_lib, T, V, n, twice):
    """The rows after it, of the same block and of the others of its cluster, wait for a walk over its entries, which may name a column twice."""
    lens = torch.full((T,), 3)
    at = [0, T // 2, T - 1]
    lens[at] = n
    gen = torch.Generator().manual_seed(7)
    order = torch.randint(0, V, (int(lens.sum()),), generator=gen)
    if not twice:
        ends = lens.cumsum(0)
        for r in at:
            order[ends[r] - n : ends[r]] = torch.randperm(V, generator=gen)[:n]
    rp = torch.zeros(T + 1, dtype=torch.int32)
    rp[1:] = lens.cumsum(0)
    va = torch.randn(order.numel(), generator=torch.Generator().manual_seed(8)).cuda()
    rp, ci = rp.cuda(), order.int().cuda()
    x = torch.randn(T, V, device="cuda", generator=_gen(V)).bfloat16()
    loss, dx = ops.distill_loss_grad(x, rp, ci, va)
    alone = ops.distill_loss(x, rp, ci, va)
    assert loss.isfinite().all() and dx.isfinite().all() and alone.isfinite().all()
    assert torch.allclose(alone, loss, rtol=1e-5, atol=1e-5)
    # the rows about the long ones, on their own, are right and the same
    some = torch.tensor(sorted({max(0, min(T - 1, r + d)) for r in at for d in (-1, 0, 1, 2)}), device="cuda")
    part_rp = torch.zeros(some.numel() + 1, dtype=torch.int32, device="cuda")
    part_rp[1:] = (rp[some + 1] - rp[some]).cumsum(0)
    take = torch.cat([torch.arange(int(rp[r]), int(rp[r + 1]), device="cuda") for r in some.tolist()])
    part = x[some], part_rp, ci[take].contiguous(), va[take].contiguous()
    check_distill(*part)
    want = ops.distill_loss_grad(*part)
    assert torch.allclose(loss[some], want[0], rtol=1e-4, atol=1e-4) and torch.allclose(dx[some].float(), want[1].float(), rtol=2.0 ** -7, atol=1e-6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("V,k", [(300, 33), (1000, 700), (1500, 256), (9001, 300), (60_000, 2000), (9001, 5000), (600_000, 3000), (3_000_000, 2500)])
@pytest.mark.parametrize("kind", ["unsorted", "twice", "same", "padded"])
def test_distill_of_many_entries_in_any_order(cuda_lib, V, k, kind, dtype):
    T = 3
    rp, ci, va = teacher(T, V, [min(k, V)] * T, 9)
    ci = ci.view(T, -1)
    n = ci.shape[1]
    if kind == "twice":
        ci[0, n // 2] = ci[0, 3]
        ci[1] = torch.randint(0, V, (n,), device="cuda", generator=_gen(10)).int()
        ci[2, : n // 2] = ci[2, n - n // 2 :]
    elif kind == "same":
        ci[0] = V - 1
        ci[1] = torch.where(torch.arange(n, device="cuda") % 3 == 0, V // 2, ci[1])
        ci[2] = torch.arange(n, device="cuda").int() // 32 * 7 % V
    elif kind == "padded":  # lists of a length that is the same for all, filled up with a column that weighs nothing
        ci[:, n // 3 :] = 0
        va.view(T, -1)[:, n // 3 :] = -float("inf")
    x = torch.randn(T, V, device="cuda", generator=_gen(V)).to(dtype)
    check_distill(x, rp, ci.flatten().contiguous(), va)
    a, b = ops.distill_loss_grad(x, rp, ci.flatten(), va), ops.distill_loss_grad(x, rp, ci.flatten(), va)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("t", [1.0, 1.2, 2.0])
@pytest.mark.parametrize("log_probs", [False, True])
@pytest.mark.parametrize("V", [300, 20000, 150_000, 600_000])
def test_distill_from_a_teacher_who_wants_what_is_masked_by_the_lowest(cuda_lib, V, log_probs, t, dtype):
    """The loss is as large as the mask, and finite: p * lowest."""
    T, k = 4, 12
    x = torch.randn(T, V, device="cuda", generator=_gen(V)).to(dtype)
    rp, ci, _ = teacher(T, V, [k] * T, 4)
    va = torch.full((T, k), -4.0, device="cuda")
    hit = ci.long().view(T, k)
    lowest = torch.finfo(dtype).min
    x[0, hit[0, 3]] = lowest
    x[1, hit[1, ::6]] = lowest  # two of equal weight: their sum before it is divided is beyond fp32
    va[2, 7] = -2.0
    x[2, hit[2, 7]] = lowest
    x[3, hit[3, 1]] = -1e38
    check_distill(x, rp, ci, va.flatten(), t, log_probs)
    assert ops.distill_loss(x, rp, ci, va.flatten(), temperature=t, log_probs=log_probs).isfinite().all()


@pytest.mark.parametrize("B", [100.0, 30000.0])
def test_route_between_groups_whose_biases_cancel(cuda_lib, B):
    """Sums of a large and a small choice are rounded at the size of what they are made of, not of what is left."""
    x = torch.randn(400_000, 8, device="cuda", generator=_gen(90))
    bias = torch.tensor([B, -B] * 4, device="cuda") + 0.25 * torch.randn(8, device="cuda", generator=_gen(91))
    _, ci, _ = ops.route(x, 2, score="sigmoid", bias=bias, groups=4, top_groups=1, group_top=2)
    want = route_f64(x, 2, bias=bias, score="sigmoid", groups=4, top_groups=1, group_top=2)[0]
    assert torch.equal(ci.long().view(-1, 2), want)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_with_groups_ranks_scores_that_round_to_the_same(cuda_lib, score):
    """Without a bias the order of the scores is that of the logits, where the scores themselves round to 1 or to 0."""
    high = [40.0, 45.0, 50.0, 41.0] if score == "sigmoid" else [0.0, -800.0, -790.0, -900.0]
    x = torch.full((3, 8), -50.0 if score == "sigmoid" else -1000.0, device="cuda")
    x[0, :4] = torch.tensor(high, device="cuda")
    x[1, 4:] = torch.tensor(high, device="cuda")
    x[2, :4] = torch.tensor(high[::-1], device="cuda")
    x[2, 4:] = torch.tensor(high, device="cuda") - 1000.0
    how = dict(score=score, groups=2, top_groups=1, group_top=2)
    _, ci, _ = ops.route(x, 2, **how)
    assert torch.equal(ci.long().view(3, 2), route_f64(x, 2, **how)[0])
    assert ci.view(3, 2).tolist() == ([[1, 2], [5, 6], [1, 2]] if score == "sigmoid" else [[0, 2], [4, 6], [1, 3]])


@pytest.mark.parametrize("Nd", [1, 6, 64, 513])
@pytest.mark.parametrize("Kd", [1, 3, 5, 70, 1000])
@pytest.mark.parametrize("nnz,kind", [(1, "one"), (31, "one"), (129, "spread"), (700, "one"), (700, "two"), (2048, "one"), (2048, "spread"), (5000, "two"), (40_000, "one")])
def test_small_product_with_the_transpose_of_crowded_columns(cuda_lib, nnz, kind, Kd, Nd):
    """All entries in one column, in two, and spread; and more of them than the operator takes this way for."""
    import ctypes as C
    from csrspmm_b200 import _lib
    M = max(1, nnz // 3)
    rp = torch.zeros(M + 1, dtype=torch.int32, device="cuda")
    rp[1:] = torch.randint(0, nnz + 1, (M,), device="cuda", generator=_gen(nnz)).sort().values
    rp[M] = nnz
    column = {"one": [Kd - 1], "two": [0, Kd // 2], "spread": list(range(Kd))}[kind]
    ci = torch.tensor(column, device="cuda", dtype=torch.int32)[torch.randint(0, len(column), (nnz,), device="cuda", generator=_gen(2))]
    va, G = torch.randn(nnz, device="cuda", generator=_gen(3)), torch.randn(M, Nd, device="cuda", generator=_gen(4))
    terms = va.double()[:, None] * G.double()[_rows(rp)]
    want, size = (torch.zeros(Kd, Nd, dtype=torch.float64, device="cuda").index_add(0, ci.long(), t) for t in (terms, terms.abs()))
    bound = (int(torch.bincount(ci.long()).max()) + 17) * U * 1.5 * size + 1e-38  # a sum in turn, of runs or of all, and the factor
    out = torch.full((Kd + 1, Nd + 3), 7.0, device="cuda")
    assert _lib.lib().csrspmm_b200_spmm_transposed(M, Kd, Nd, nnz, rp.data_ptr(), ci.data_ptr(), va.data_ptr(), G.data_ptr(), Nd, 1.5, out.data_ptr(),
                                                   Nd + 3, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    assert ((out[:Kd, :Nd].double() - 1.5 * want).abs() <= bound).all() and (out[:Kd, Nd:] == 7).all() and (out[Kd] == 7).all()
    again = torch.ops.csrspmm_b200.spmm_transposed(rp, ci, va, G, Kd, 1.5)
    assert ((again.double() - 1.5 * want).abs() <= bound).all()
    assert torch.equal(again, torch.ops.csrspmm_b200.spmm_transposed(rp, ci, va, G, Kd, 1.5))


def test_the_64_bit_exponential_and_reciprocal_of_the_choice(cuda_lib):
    """Over their whole range, against long double; the program states the bounds."""
    import subprocess
    from pathlib import Path
    exe = Path(__file__).parent / "cpp" / "_bin" / "test_route_math"
    assert exe.exists(), "tests/cpp/_bin/test_route_math not built (python -m csrspmm_b200.build)"
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout + run.stderr
