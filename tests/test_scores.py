"""Routing, the gradient for stored values and distillation: what is refused, and what needs no GPU."""
import ctypes as C

import pytest
import torch

from csrspmm_b200 import _lib, build, ops, torch_library  # noqa: F401

P = 4096  # an address that nothing reads: every call here is refused, or launches into a runtime that runs no kernels


def _route(**kw):
    base = dict(struct_size=C.sizeof(_lib.RouteArgs), T=8, E=64, k=4, scores=P, ld=64, score_type=0, score=0, bias=None, groups=8, top_groups=4,
                group_top=2, renormalize=1, scale=1.0)
    return _lib.RouteArgs(**{**base, **kw})


def _distill(**kw):
    base = dict(struct_size=C.sizeof(_lib.DistillArgs), T=8, V=100, logit_type=2, logits=P, ld=100, nnz=20, row_ptr=P, col_idx=P, values=P,
                temperature=1.0, log_probs=0)
    return _lib.DistillArgs(**{**base, **kw})


BAD_ROUTE = [dict(struct_size=8), dict(T=-1), dict(E=0, ld=0), dict(E=1025, ld=1025, groups=1, top_groups=1, group_top=1), dict(score_type=3),
             dict(score_type=-1), dict(score=2), dict(score=-1), dict(groups=0), dict(groups=7), dict(groups=64, top_groups=64, group_top=1),
             dict(top_groups=0), dict(top_groups=9), dict(group_top=0), dict(group_top=3), dict(groups=64, top_groups=1, group_top=2), dict(k=0),
             dict(k=33), dict(k=32, top_groups=1), dict(ld=63), dict(scale=float("inf")), dict(scale=float("nan")), dict(scores=None),
             dict(T=1 << 30, k=4)]
BAD_DISTILL = [dict(struct_size=0), dict(T=-1), dict(V=-1), dict(ld=99), dict(nnz=-1), dict(nnz=1 << 31), dict(logit_type=3), dict(logit_type=-1),
               dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan")),
               dict(temperature=1e-39), dict(V=0, ld=0), dict(logits=None), dict(row_ptr=None), dict(col_idx=None), dict(values=None)]


@pytest.mark.parametrize("change", BAD_ROUTE, ids=str)
def test_bad_routing_is_refused_before_any_cuda_call(change):
    L, a = _lib.lib(), _route(**change)
    assert L.csrspmm_b200_route(C.byref(a), P, P, P, None) == _lib.ERR_BAD_ARG
    assert L.csrspmm_b200_last_error().startswith(b"route: ")
    assert L.csrspmm_b200_route_backward(C.byref(a), P, P, P, 1, P, 2000, None) == _lib.ERR_BAD_ARG


@pytest.mark.parametrize("change", BAD_DISTILL, ids=str)
def test_bad_distillation_is_refused_before_any_cuda_call(change):
    L, a = _lib.lib(), _distill(**change)
    assert L.csrspmm_b200_distill(C.byref(a), P, P, None) == _lib.ERR_BAD_ARG
    assert L.csrspmm_b200_last_error().startswith(b"distill: ")
    assert L.csrspmm_b200_distill_backward(C.byref(a), P, P, 1, P, 100, None) == _lib.ERR_BAD_ARG
    assert L.csrspmm_b200_distill_grad(C.byref(a), P, 1, P, P, 100, None) == _lib.ERR_BAD_ARG


@pytest.mark.parametrize("t", [1e20, 2e19, 1e-20, 1e-37])
def test_temperatures_whose_square_is_not_in_fp32_are_refused(t):
    """The loss is t^2 times what is left of sums of numbers of size 1."""
    L, a = _lib.lib(), _distill(temperature=t)
    assert L.csrspmm_b200_distill(C.byref(a), P, P, None) == _lib.ERR_BAD_ARG
    assert b"square of the temperature" in L.csrspmm_b200_last_error()
    assert L.csrspmm_b200_distill_backward(C.byref(a), P, P, 1, P, 100, None) == _lib.ERR_BAD_ARG
    assert L.csrspmm_b200_distill_grad(C.byref(a), P, 1, P, P, 100, None) == _lib.ERR_BAD_ARG


def test_missing_outputs_are_refused():
    L, r, d = _lib.lib(), _route(), _distill()
    bad = _lib.ERR_BAD_ARG
    for out in ((None, P, P), (P, None, P), (P, P, None)):
        assert L.csrspmm_b200_route(C.byref(r), *out, None) == bad
    for arrays in ((None, P, P, 1, P), (P, None, P, 1, P), (P, P, None, 1, P), (P, P, P, 1, None)):
        assert L.csrspmm_b200_route_backward(C.byref(r), *arrays, 64, None) == bad
    assert L.csrspmm_b200_route_backward(C.byref(r), P, P, P, 1, P, 63, None) == bad
    assert L.csrspmm_b200_route(None, P, P, P, None) == bad and L.csrspmm_b200_distill(None, P, P, None) == bad
    assert L.csrspmm_b200_distill(C.byref(d), None, P, None) == bad and L.csrspmm_b200_distill(C.byref(d), P, P + 8, None) == bad
    assert L.csrspmm_b200_distill_backward(C.byref(d), P + 8, P, 1, P, 100, None) == bad
    assert L.csrspmm_b200_distill_backward(C.byref(d), P, P, 1, P, 99, None) == bad
    assert L.csrspmm_b200_distill_grad(C.byref(d), None, 1, P, P, 100, None) == bad
    assert L.csrspmm_b200_distill_grad(C.byref(d), P, 1, P, None, 100, None) == bad


@pytest.mark.parametrize("args", [(-1, 4, 4, 5), (4, -1, 4, 5), (4, 4, -1, 5), (4, 4, 4, -1), (4, 4, 4, 1 << 31), (0, 4, 4, 5), (4, 0, 4, 5)], ids=str)
def test_bad_sizes_of_the_sampled_product_are_refused(args):
    assert _lib.lib().csrspmm_b200_sddmm(*args, P, P, P, 4, P, 4, 1.0, P, None) == _lib.ERR_BAD_ARG


def test_bad_arguments_of_the_small_product_with_the_transpose_are_refused():
    L = _lib.lib()
    good = [4, 4, 4, 5, P, P, P, P, 4, 1.0, P, 4, None]
    for at, value in ((0, -1), (1, -1), (2, -1), (3, -1), (3, 1 << 31), (0, 0), (4, None), (5, None), (6, None), (7, None), (8, 3), (10, None), (11, 3)):
        args = list(good)
        args[at] = value
        assert L.csrspmm_b200_spmm_transposed(*args) == _lib.ERR_BAD_ARG, (at, value)
    assert L.csrspmm_b200_spmm_transposed(0, 0, 4, 0, None, None, None, None, 4, 1.0, None, 4, None) == 0
    assert L.csrspmm_b200_spmm_transposed_pays(100, 64, 500) == 1 and L.csrspmm_b200_spmm_transposed_pays(1 << 20, 64, 1 << 24) == 0
    assert L.csrspmm_b200_spmm_transposed_pays(-1, 64, 500) == 0


def test_the_small_product_with_the_transpose_is_taken_only_where_no_column_can_be_crowded():
    pays = _lib.lib().csrspmm_b200_spmm_transposed_pays
    for Kd, Nd, nnz in ((64, 512, 131_072), (32, 512, 524_288), (64, 512, 262_144), (1, 512, 1 << 24), (1, 1, 1 << 24), (8, 64, 32_768), (200, 64, 2049),
                        (2048, 512, 2048), (1024, 513, 1024), (1 << 30, 1 << 30, 2048), (2 ** 31 - 1, 2 ** 31 - 1, 1)):
        assert pays(Kd, Nd, nnz) == 0, (Kd, Nd, nnz)
    for Kd, Nd, nnz in ((1, 1, 0), (8, 512, 2048), (64, 512, 2048), (1024, 512, 1024), (512, 2048, 512), (2048, 64, 2048), (256, 513, 512)):
        assert pays(Kd, Nd, nnz) == 1, (Kd, Nd, nnz)


def test_bad_pointers_of_the_sampled_product_are_refused():
    good = [4, 4, 4, 5, P, P, P, 4, P, 4, 1.0, P, None]
    for at, value in ((4, None), (5, None), (6, None), (7, 3), (8, None), (9, 3), (11, None)):
        args = list(good)
        args[at] = value
        assert _lib.lib().csrspmm_b200_sddmm(*args) == _lib.ERR_BAD_ARG


def test_tensors_on_the_host_are_refused():
    rp, ci, va = torch.zeros(5, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(0)
    with pytest.raises(RuntimeError, match="logits must be a 2-D CUDA tensor"):
        ops.route(torch.zeros(4, 8), 2)
    with pytest.raises(RuntimeError, match="logits must be a 2-D CUDA tensor"):
        ops.distill_loss(torch.zeros(4, 8), rp, ci, va)
    with pytest.raises(RuntimeError, match="logits must be a 2-D CUDA tensor"):
        ops.distill_loss_grad(torch.zeros(4, 8), rp, ci, va)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.sddmm(rp, ci, torch.zeros(4, 3), torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        ops.weighted_spmm(rp, ci, va, torch.zeros(2, 3))


def test_tangents_are_refused_not_dropped():
    import torch.autograd.forward_ad as fwAD
    rp, ci, va = torch.zeros(5, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(0)
    with fwAD.dual_level():
        x = fwAD.make_dual(torch.zeros(4, 8), torch.ones(4, 8))
        for call in (lambda: ops.route(x, 2), lambda: ops.distill_loss(x, rp, ci, va), lambda: ops.weighted_spmm(rp, ci, va, x)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_tangents_are_refused_where_no_derivative_is_recorded():
    import torch.autograd.forward_ad as fwAD
    O = torch.ops.csrspmm_b200
    rp, ci, va = torch.zeros(5, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(0)
    with fwAD.dual_level():
        x, w, v = (fwAD.make_dual(torch.zeros(*s), torch.ones(*s)) for s in ((4, 8), (4,), (0,)))
        flat, one = torch.zeros(4, 8), torch.ones(4)
        for call in (lambda: ops.sddmm(rp, ci, x, flat), lambda: ops.sddmm(rp, ci, flat, x), lambda: O.sddmm(rp, ci, x, flat, 1.0),
                     lambda: O.sddmm(rp, ci, flat, x, 1.0), lambda: ops.distill_loss_grad(x, rp, ci, va), lambda: ops.distill_loss_grad(flat, rp, ci, va, w),
                     lambda: ops.distill_loss_grad(flat, rp, ci, v), lambda: O.distill_loss_grad(x, rp, ci, va, one, 1.0, False),
                     lambda: O.distill_loss_grad(flat, rp, ci, va, w, 1.0, False), lambda: O.distill_loss_grad(flat, rp, ci, v, one, 1.0, False),
                     lambda: O.route(x, 2, None, "softmax", 1, 1, 1, True, 1.0), lambda: O.distill_loss(x, rp, ci, va, 1.0, False),
                     lambda: O.weighted_spmm(rp, ci, v, flat, 1.0)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_gradients_for_a_teacher_are_refused():
    rp, ci, va = torch.zeros(5, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(0, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient for the teacher"):
        ops.distill_loss(torch.zeros(4, 8, requires_grad=True), rp, ci, va)


def test_the_operators_trace_without_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode
    O = torch.ops.csrspmm_b200
    with FakeTensorMode():
        x = torch.empty(6, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        rp, ci, va = O.route(x, 4, None, "softmax", 4, 2, 1, True, 1.0)
        assert (rp.shape, ci.shape, va.shape) == ((7,), (24,), (24,)) and (rp.dtype, ci.dtype, va.dtype) == (torch.int32, torch.int32, torch.float32)
        assert va.requires_grad and not rp.requires_grad
        dx = O.route_backward(torch.empty_like(va), x.detach(), ci, va.detach(), 4, "softmax", True, 1.0)  # the engine itself wants a GPU
        assert dx.shape == x.shape and dx.dtype == x.dtype
        B = torch.empty(16, 5, device="cuda", requires_grad=True)
        out = O.weighted_spmm(rp, ci, va.detach().requires_grad_(True), B, 1.0)
        assert out.shape == (6, 5) and out.requires_grad
        assert O.sddmm(rp, ci, out.detach(), B.detach(), 1.0).shape == (24,)
        loss = O.distill_loss(x, rp, ci, va.detach(), 1.0, False)
        assert loss.shape == (6,) and loss.dtype == torch.float32
        assert loss.requires_grad
        loss, stats = O.distill_with_stats(x.detach(), rp, ci, va.detach(), 1.0, False)
        dx = O.distill_backward(loss, x.detach(), rp, ci, va.detach(), stats, 1.0, False)
        assert dx.shape == x.shape and dx.dtype == x.dtype
        loss, dx = O.distill_loss_grad(x.detach(), rp, ci, va.detach(), loss.detach(), 1.0, True)
        assert loss.shape == (6,) and dx.dtype == torch.bfloat16


@pytest.fixture(scope="module")
def fake():
    L = C.CDLL(str(build.build_fake_runtime()))
    for name in ("fake_kernels", "fake_launched"):
        getattr(L, name).restype = C.c_size_t
    L.fake_reset.argtypes = [C.c_long]
    for name in ("route", "route_backward", "sddmm", "spmm_transposed", "distill", "distill_backward", "distill_grad"):
        getattr(L, "csrspmm_b200_" + name).argtypes = getattr(_lib.lib(), "csrspmm_b200_" + name).argtypes
    return L


def _names(function):
    text = C.create_string_buffer(function(None))
    function(text)
    return set(text.value.decode().split("\n")) - {""}


def test_nothing_is_compiled_that_no_call_launches(fake):
    fake.fake_reset(0)
    for kind in range(3):
        for E in (2, 64, 65, 128, 129, 256, 257, 512, 513, 1024):
            for groups, bias in ((1, None), (1, P), (2, None)):
                a = _route(E=E, k=1, ld=E, score_type=kind, groups=groups if E % 2 == 0 else 1, top_groups=1, group_top=1, bias=bias)
                assert fake.csrspmm_b200_route(C.byref(a), P, P, P, None) == 0
                assert fake.csrspmm_b200_route_backward(C.byref(a), P, P, P, 1, P, E, None) == 0
        for T in (1, 8, 4000):
            for V in (1, 1000, 6000, 8192, 8193, 15000, 30000, 70000, 300000, 600_000, 3_000_000):
                d = _distill(T=T, V=V, ld=V, logit_type=kind)
                assert fake.csrspmm_b200_distill(C.byref(d), P, P, None) == 0
                assert fake.csrspmm_b200_distill_grad(C.byref(d), P, 1, P, P, V, None) == 0
                assert fake.csrspmm_b200_distill_backward(C.byref(d), P, P, 1, P, V, None) == 0
    for Nd in (1, 2, 3, 8, 9, 16, 17, 18, 33, 34, 50, 64, 65, 90, 100, 129, 130, 200, 256, 257, 258, 512, 513, 514, 1000, 1024):
        assert fake.csrspmm_b200_sddmm(100, 50, Nd, 1000, P, P, P, Nd, P, Nd, 1.0, P, None) == 0
        assert fake.csrspmm_b200_spmm_transposed(100, 50, Nd, 1000, P, P, P, P, Nd, 1.0, P, Nd, None) == 0
    every = {k for k in _names(fake.fake_kernels) if any(w in k for w in ("route_", "sddmm_", "distill_", "spmm_transposed"))}
    assert every and sorted(every - _names(fake.fake_launched)) == []


def test_rows_of_more_entries_than_a_list_holds_take_the_kernel_in_which_all_warps_walk_over_them(fake):
    for T, V in ((1000, 100_000), (20_000, 6000)):
        for per_row, ring in ((64, True), (256, True), (257, False), (2048, False)):
            a = _distill(T=T, V=V, ld=V, nnz=T * per_row)
            fake.fake_reset(0)
            assert fake.csrspmm_b200_distill(C.byref(a), P, P, None) == 0 and fake.csrspmm_b200_distill_grad(C.byref(a), P, 1, P, P, V, None) == 0
            names = _names(fake.fake_launched)
            assert len(names) == 2 and all(("distill_ring_kernel" if ring else "distill_long_kernel") in n for n in names)


def test_a_failed_launch_is_reported(fake):
    for run in (lambda: fake.csrspmm_b200_route(C.byref(_route()), P, P, P, None),
                lambda: fake.csrspmm_b200_route_backward(C.byref(_route()), P, P, P, 1, P, 64, None),
                lambda: fake.csrspmm_b200_route(C.byref(_route(E=1024, ld=1024)), P, P, P, None),
                lambda: fake.csrspmm_b200_route(C.byref(_route(T=0)), C.addressof(C.create_string_buffer(16)), P, P, None),
                lambda: fake.csrspmm_b200_sddmm(4, 4, 4, 5, P, P, P, 4, P, 4, 1.0, P, None),
                lambda: fake.csrspmm_b200_spmm_transposed(4, 4, 4, 5, P, P, P, P, 4, 1.0, P, 4, None),
                lambda: fake.csrspmm_b200_distill(C.byref(_distill()), P, P, None),
                lambda: fake.csrspmm_b200_distill_backward(C.byref(_distill()), P, P, 1, P, 100, None),
                lambda: fake.csrspmm_b200_distill_grad(C.byref(_distill()), P, 1, P, P, 100, None)):
        fake.fake_reset(1)
        assert run() == _lib.ERR_CUDA
        fake.fake_reset(0)
        assert run() == 0


def test_batches_in_which_a_row_may_hold_very_many_entries_take_the_kernel_without_waits(fake):
    for nnz, ring in ((1 << 25, True), ((1 << 25) + 1, False)):
        a = _distill(T=200_000, V=100_000, ld=100_000, nnz=nnz)
        for call in (lambda: fake.csrspmm_b200_distill(C.byref(a), P, P, None), lambda: fake.csrspmm_b200_distill_grad(C.byref(a), P, 1, P, P, 100_000, None)):
            fake.fake_reset(0)
            assert call() == 0
            (name,) = _names(fake.fake_launched)
            assert ("distill_ring_kernel" in name) == ring and ("distill_long_kernel" in name) != ring
