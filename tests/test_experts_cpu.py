"""Refusals of the expert and sandwich-norm entry points, without a GPU: the
device check is replaced so CPU tensors pass it, and the library must not be
reached."""
from __future__ import annotations

import pytest
import torch

F16, F32, I32 = torch.float16, torch.float32, torch.int32


class _Unreached(Exception):
    pass


@pytest.fixture
def k(pkg, monkeypatch):
    kern = pkg.kernels

    def device(t, name):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        return t.device

    def load():
        raise _Unreached

    monkeypatch.setattr(kern, "_cuda_tensor", device)
    monkeypatch.setattr(kern._lib, "load", load)
    return kern


def test_cpu_tensors_are_refused(pkg):
    kern = pkg.kernels
    with pytest.raises(ValueError, match="CUDA"):
        kern.route_experts(torch.zeros(2, 4), 1)
    with pytest.raises(ValueError, match="CUDA"):
        kern.sandwich_norm(torch.zeros(2, 8), torch.zeros(2, 8, dtype=F16), torch.ones(8))
    with pytest.raises(TypeError):
        kern.route_experts([[1.0]], 1)


def test_plan_and_workspace_sizes(pkg):
    lib = pkg._lib.load()
    assert lib.tj_expert_plan_ints(0, 2, 8) == 9 + 8
    assert lib.tj_expert_plan_ints(64, 2, 8) == 9 + 256 + 8
    assert lib.tj_expert_plan_ints(65, 2, 8) == 9 + 260 + 16
    assert lib.tj_expert_plan_ints(100000, 4, 64) == 65 + 800000 + 148 * 64
    assert lib.tj_expert_plan_ints(-1, 2, 8) == 0 and lib.tj_expert_plan_ints(1, 0, 8) == 0
    assert lib.tj_expert_ffn_workspace_bytes(10, 2, 4, 64, 128) == 20 * 256 + 20 * 256
    assert lib.tj_expert_ffn_workspace_bytes(10, 0, 4, 64, 128) == 0
    assert lib.tj_gemm_experts_workspace_bytes(64, 2, 4, 64, 1) == 0  # 32 rows per expert: gathered by the kernel
    assert lib.tj_gemm_experts_workspace_bytes(65, 2, 4, 64, 1) == 130 * 128
    assert lib.tj_gemm_experts_workspace_bytes(65, 2, 4, 64, 0) == 0


@pytest.mark.parametrize("kw,error", [
    (dict(logits=torch.zeros(4, 8, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(4)), ValueError),
    (dict(logits=torch.zeros(8, 4).t()), ValueError),
    (dict(top_k=0), ValueError),
    (dict(top_k=9), ValueError),
    (dict(logits=torch.zeros(4, 64), top_k=33), ValueError),
    (dict(scoring="max"), ValueError),
    (dict(bias=torch.zeros(7)), ValueError),
    (dict(bias=torch.zeros(8, dtype=F16)), TypeError),
    (dict(row_count=torch.zeros(2, dtype=I32)), ValueError),
    (dict(row_count=torch.zeros(1, dtype=torch.int64)), TypeError),
    (dict(logits=torch.zeros(4, 8, requires_grad=True)), RuntimeError),
])
def test_route_refusals(k, kw, error):
    args = dict(logits=torch.zeros(4, 8), top_k=2)
    with pytest.raises(_Unreached):
        k.route_experts(**args)
    args.update(kw)
    with pytest.raises(error):
        k.route_experts(**args)


def test_no_grad_is_allowed(k):
    with torch.no_grad(), pytest.raises(_Unreached):
        k.route_experts(torch.zeros(4, 8, requires_grad=True), 2)


def _routing(k, rows=4, top_k=2, E=3):
    return k.ExpertRouting(torch.zeros(rows, top_k, dtype=I32), torch.zeros(rows, top_k),
                           torch.zeros(E + 1 + 3 * rows * top_k, dtype=I32), E)


@pytest.mark.parametrize("args,error", [
    ((torch.zeros(4, 2), torch.zeros(4, 2), 3), TypeError),
    ((torch.zeros(4, dtype=I32), torch.zeros(4), 3), ValueError),
    ((torch.zeros(4, 33, dtype=I32), torch.zeros(4, 33), 3), ValueError),
    ((torch.zeros(4, 2, dtype=I32), torch.zeros(4, 1), 3), ValueError),
    ((torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), 0), ValueError),
    ((torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), 513), ValueError),
])
def test_plan_refusals(k, args, error):
    with pytest.raises(error):
        k.expert_plan(*args)


@pytest.mark.parametrize("kw,error", [
    (dict(a=torch.zeros(4, 16)), TypeError),
    (dict(a=torch.zeros(5, 16, dtype=F16)), ValueError),
    (dict(a=torch.zeros(4, 24, dtype=F16)), ValueError),
    (dict(w_in=torch.zeros(3, 32, 16, dtype=torch.bfloat16)), TypeError),
    (dict(w_in=torch.zeros(2, 32, 16, dtype=F16)), ValueError),
    (dict(w_out=torch.zeros(3, 16, 24, dtype=F16)), ValueError),
    (dict(w_out=torch.zeros(3, 32, 16, dtype=F16).transpose(1, 2)), ValueError),
    (dict(b_in=torch.zeros(3, 16)), ValueError),
    (dict(b_out=torch.zeros(3, 16, dtype=F16)), TypeError),
    (dict(routing=None), TypeError),
    (dict(w_in=torch.zeros(3, 32, 16, dtype=F16, requires_grad=True)), RuntimeError),
])
def test_ffn_refusals(k, kw, error):
    args = dict(a=torch.zeros(4, 16, dtype=F16), w_in=torch.zeros(3, 32, 16, dtype=F16), b_in=torch.zeros(3, 32),
                w_out=torch.zeros(3, 16, 32, dtype=F16), b_out=None, routing=_routing(k))
    with pytest.raises(_Unreached):
        k.expert_ffn(**args)
    args.update(kw)
    with pytest.raises(error):
        k.expert_ffn(**args)


def test_gemm_and_combine_refusals(k):
    r = _routing(k)
    w = torch.zeros(3, 32, 16, dtype=F16)
    for a, gather in ((torch.zeros(4, 16, dtype=F16), True), (torch.zeros(8, 16, dtype=F16), False)):
        with pytest.raises(_Unreached):
            k.gemm_experts(a, w, None, r, gather=gather)
        with pytest.raises(ValueError):
            k.gemm_experts(a, w, None, r, gather=not gather)
        with pytest.raises(ValueError):
            k.gemm_experts(a, w, torch.zeros(3, 16), r, gather=gather)
    with pytest.raises(_Unreached):
        k.expert_combine(torch.zeros(8, 16, dtype=F16), r)
    with pytest.raises(ValueError):
        k.expert_combine(torch.zeros(4, 16, dtype=F16), r)
    with pytest.raises(TypeError):
        k.expert_combine(torch.zeros(8, 16), r)
    with pytest.raises(TypeError):
        k.expert_combine(torch.zeros(8, 16, dtype=F16), object())


@pytest.mark.parametrize("kw,error", [
    (dict(x=torch.zeros(4, 16, dtype=F16)), TypeError),
    (dict(x=torch.zeros(3, 16)), ValueError),
    (dict(x=torch.zeros(64)), ValueError),
    (dict(branch=torch.zeros(4, 16)), TypeError),
    (dict(branch=torch.zeros(4, 8, dtype=F16)), ValueError),
    (dict(pre_gamma=torch.ones(8)), ValueError),
    (dict(pre_gamma=None), ValueError),
    (dict(pre_beta=torch.ones(16, dtype=F16)), TypeError),
    (dict(post_beta=torch.ones(16)), ValueError),
    (dict(kind="batch"), ValueError),
    (dict(gate_act="relu"), ValueError),
    (dict(gate=torch.zeros(8)), ValueError),
    (dict(gate=torch.zeros(16, dtype=F16)), TypeError),
    (dict(gate=torch.zeros(4, 16, dtype=torch.bfloat16)), TypeError),
    (dict(gate=torch.zeros(0, 16)), ValueError),
    (dict(gate=torch.zeros(1, 16), rows_per_gate=3), ValueError),
    (dict(gate=torch.zeros(4, 16), rows_per_gate=0), ValueError),
    (dict(gate=torch.zeros(4, 16), gate_map=torch.zeros(3, dtype=I32)), ValueError),
    (dict(row_map=torch.zeros(4)), TypeError),
    (dict(row_map=torch.zeros(5, dtype=I32)), ValueError),
    (dict(routing="r"), TypeError),
    (dict(gate=torch.zeros(16, requires_grad=True)), RuntimeError),
])
def test_sandwich_refusals(k, kw, error):
    args = dict(x=torch.zeros(4, 16), branch=torch.zeros(4, 16, dtype=F16), pre_gamma=torch.ones(16))
    with pytest.raises(_Unreached):
        k.sandwich_norm(**args)
    args.update(kw)
    with pytest.raises(error):
        k.sandwich_norm(**args)


def test_outputs_that_share_memory_are_refused(k):
    r = _routing(k, rows=4, top_k=1)
    a = torch.zeros(4, 16, dtype=F16)
    with pytest.raises(ValueError, match="share"):
        k.gemm_experts(a, torch.zeros(3, 16, 16, dtype=F16), None, r, gather=False, out=a)
    with pytest.raises(ValueError, match="share"):
        k.expert_combine(a, r, out=a)
    big = torch.zeros(5, 16)
    x, gamma = big[:4], torch.ones(16)
    with pytest.raises(_Unreached):
        k.sandwich_norm(x, a, gamma, sum_out=x, out=a)
    for kw in (dict(sum_out=big[1:]), dict(sum_out=x, row_map=torch.zeros(4, dtype=I32)), dict(out=a, routing=r)):
        with pytest.raises(ValueError, match="share"):
            k.sandwich_norm(x, a, gamma, **kw)
    half = torch.zeros(4, 32, dtype=F16)
    with pytest.raises(ValueError, match="share"):
        k.sandwich_norm(half.view(torch.float32), a, gamma, out=half.view(8, 16)[:4])


@pytest.mark.parametrize("experts,weights,plan,error", [
    (torch.zeros(4, 2, dtype=I32), torch.zeros(4, 1), torch.zeros(20, dtype=I32), ValueError),
    (torch.zeros(4, 2), torch.zeros(4, 2), torch.zeros(20, dtype=I32), TypeError),
    (torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), torch.zeros(19, dtype=I32), ValueError),
    (torch.zeros(8, dtype=I32), torch.zeros(8), torch.zeros(20, dtype=I32), ValueError),
])
def test_routing_buffers_are_checked(k, experts, weights, plan, error):
    k.ExpertRouting(torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), torch.zeros(20, dtype=I32), 3)
    with pytest.raises(error):
        k.ExpertRouting(experts, weights, plan, 3)


def test_weights_of_the_routing_that_need_a_gradient_are_refused(k):
    """A routing may be made of weights that need one; whatever sums with them refuses."""
    r = k.ExpertRouting(torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2, requires_grad=True),
                        torch.zeros(4 + 24, dtype=I32), 3)
    a, y = torch.zeros(4, 16, dtype=F16), torch.zeros(8, 16, dtype=F16)
    w_in, w_out = torch.zeros(3, 32, 16, dtype=F16), torch.zeros(3, 16, 32, dtype=F16)
    calls = (lambda: k.expert_ffn(a, w_in, None, w_out, None, r), lambda: k.expert_combine(y, r),
             lambda: k.sandwich_norm(torch.zeros(4, 16), y, torch.ones(16), routing=r))
    for call in calls:
        with pytest.raises(RuntimeError, match="autograd"):
            call()
        with torch.no_grad(), pytest.raises(_Unreached):
            call()


def test_forward_mode_tangents_are_refused(k):
    from torch.autograd import forward_ad

    def dual(*shape, dtype=F32):
        return forward_ad.make_dual(torch.zeros(*shape, dtype=dtype), torch.ones(*shape, dtype=dtype))

    r = _routing(k)
    a, y = torch.zeros(4, 16, dtype=F16), torch.zeros(8, 16, dtype=F16)
    w_in, w_out = torch.zeros(3, 32, 16, dtype=F16), torch.zeros(3, 16, 32, dtype=F16)
    with forward_ad.dual_level():
        with pytest.raises(_Unreached):  # no tangent: nothing to lose
            k.route_experts(torch.zeros(4, 8), 2)
        calls = (lambda: k.route_experts(dual(4, 8), 2),
                 lambda: k.route_experts(torch.zeros(4, 8), 2, bias=dual(8)),
                 lambda: k.expert_plan(torch.zeros(4, 2, dtype=I32), dual(4, 2), 3),
                 lambda: k.gemm_experts(a, dual(3, 32, 16, dtype=F16), None, r, gather=True),
                 lambda: k.expert_combine(dual(8, 16, dtype=F16), r),
                 lambda: k.expert_ffn(dual(4, 16, dtype=F16), w_in, None, w_out, None, r),
                 lambda: k.sandwich_norm(dual(4, 16), a, torch.ones(16)),
                 lambda: k.sandwich_norm(torch.zeros(4, 16), y, dual(16), routing=r))
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()


def _views(nbytes):
    """Views of one buffer: floats [4, 16], halves [4, 16], ints and vectors over the same bytes."""
    raw = torch.zeros(nbytes, dtype=torch.uint8)
    return lambda dtype, *shape: raw[: torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()].view(dtype).view(shape)


@pytest.mark.parametrize("out", ["sum_out", "out"])
@pytest.mark.parametrize("name,dtype,shape", [
    ("gate", F32, (2, 16)), ("gate", F32, (16,)), ("gate", F16, (4, 16)), ("pre_gamma", F32, (16,)), ("pre_beta", F32, (16,)),
    ("post_gamma", F32, (16,)), ("post_beta", F32, (16,)), ("row_map", I32, (4,)), ("gate_map", I32, (4,)),
    ("row_count", I32, (1,))])
def test_sandwich_outputs_over_other_inputs_are_refused(k, out, name, dtype, shape):
    """Another row's output would be written over what this row still reads."""
    view = _views(256)
    args = dict(x=torch.zeros(4, 16), branch=torch.zeros(4, 16, dtype=F16), pre_gamma=torch.ones(16))
    args[name] = view(dtype, *shape)
    if name == "post_beta":
        args["post_gamma"] = torch.ones(16)
    if name == "gate" and len(shape) == 2:
        args["rows_per_gate"] = 4 // shape[0]
    if name == "gate_map":
        args["gate"] = torch.zeros(4, 16)
    with pytest.raises(_Unreached):
        k.sandwich_norm(**args)
    args[out] = view(F32 if out == "sum_out" else F16, 4, 16)
    with pytest.raises(ValueError, match="share memory with " + name):
        k.sandwich_norm(**args)


@pytest.mark.parametrize("name", ["weights", "plan", "row_count"])
def test_outputs_over_the_routing_are_refused(k, name):
    view = _views(512)
    parts = dict(experts=torch.zeros(4, 2, dtype=I32), weights=torch.zeros(4, 2), plan=torch.zeros(28, dtype=I32),
                 row_count=torch.zeros(1, dtype=I32))
    parts[name] = view(parts[name].dtype, *parts[name].shape)
    r = k.ExpertRouting(parts["experts"], parts["weights"], parts["plan"], 3, parts["row_count"])
    a, y, out = torch.zeros(4, 16, dtype=F16), torch.zeros(8, 16, dtype=F16), view(F16, 4, 16)
    w_in, w_out = torch.zeros(3, 32, 16, dtype=F16), torch.zeros(3, 16, 32, dtype=F16)
    calls = [lambda: k.expert_combine(y, r, out=out), lambda: k.expert_ffn(a, w_in, None, w_out, None, r, out=out),
             lambda: k.sandwich_norm(torch.zeros(4, 16), y, torch.ones(16), routing=r, out=out),
             lambda: k.sandwich_norm(torch.zeros(4, 16), y, torch.ones(16), routing=r, sum_out=view(F32, 4, 16))]
    if name == "plan":
        calls.append(lambda: k.gemm_experts(y, w_in[:, :16].contiguous(), None, r, gather=False, out=view(F16, 8, 16)))
    for call in calls:
        with pytest.raises(ValueError, match="share"):
            call()


def test_ffn_output_over_weights_is_refused_and_over_a_is_not(k):
    r = _routing(k)
    a = torch.zeros(4, 16, dtype=F16)
    w_in, w_out = torch.zeros(3, 32, 16, dtype=F16), torch.zeros(3, 16, 32, dtype=F16)
    b_out = torch.zeros(3, 16)
    with pytest.raises(_Unreached):
        k.expert_ffn(a, w_in, None, w_out, b_out, r, out=a)
    for out in (w_in[0, :4], w_out.view(-1)[:64].view(4, 16), b_out.view(F16).view(-1)[:64].view(4, 16)):
        with pytest.raises(ValueError, match="share"):
            k.expert_ffn(a, w_in, None, w_out, b_out, r, out=out)


def test_sizes_past_32_bits_are_refused(k):
    """Not taken modulo 2^32: tensors without storage stand for the large ones."""
    many = 2**32 + 5

    def meta(*shape, dtype=F32):
        return torch.empty(*shape, dtype=dtype, device="meta")

    r = _routing(k)
    rm = k.ExpertRouting(meta(4, 2, dtype=I32), meta(4, 2), meta(28, dtype=I32), 3)
    calls = [lambda kw=kw: k.route_experts(torch.zeros(4, 8), 2, **kw)
             for kw in (dict(num_groups=2**32 + 2), dict(num_groups=2, top_groups=2**32 + 1),
                        dict(num_groups=2, group_score_top=2**32 + 1))]
    calls += [lambda: k.route_experts(meta(many, 1), 1),
              lambda: k.expert_plan(meta(many, 1, dtype=I32), meta(many, 1), 3),
              lambda: k.ExpertRouting(meta(many, 1, dtype=I32), meta(many, 1), meta(4 * many, dtype=I32), 3),
              lambda: k.ExpertRouting(r.experts, r.weights, r.plan, -(2**32) + 3),
              lambda: k.sandwich_norm(meta(many, 1), meta(many, 1, dtype=F16), meta(1)),
              lambda: k.sandwich_norm(meta(many, 1), meta(5, 1, dtype=F16), meta(1)),
              lambda: k.sandwich_norm(torch.zeros(4, 16), torch.zeros(4, 16, dtype=F16), torch.ones(16),
                                      gate=torch.zeros(1, 16), rows_per_gate=2**32 + 4),
              lambda: k.gemm_experts(meta(4, many, dtype=F16), meta(3, 8, many, dtype=F16), None, rm, gather=True),
              lambda: k.gemm_experts(meta(4, 8, dtype=F16), meta(3, many, 8, dtype=F16), None, rm, gather=True),
              lambda: k.expert_combine(meta(8, many, dtype=F16), rm),
              lambda: k.expert_ffn(meta(4, 8, dtype=F16), meta(3, many, 8, dtype=F16), None, meta(3, 8, many, dtype=F16), None,
                                   rm)]
    for call in calls:
        with pytest.raises(ValueError, match="32 bits"):
            call()
