"""window_attention and prefix_attention without a GPU: tracing, plans, sharding roles and refusals."""
import ctypes

import pytest
import torch

import conductor
from cache_attention_ref import reference
from conductor.compiler import loader
from conductor.compiler.executor import attention_view_ok, make_descriptors
from conductor.compiler.jit_compiler import ChoreoJITCompiler
from conductor.compiler.sharding import batch_inputs
from conductor.utils.exceptions import ConductorError, DeviceError, UnsupportedOperationError
from conductor_b200.codegen import kernel_templates as kt
from conductor_b200.codegen.operator_registry import Template


def compile_plan(fn, *args):
    """The plan the backend makes of fn (nothing runs)."""
    torch._dynamo.reset()
    box = []

    def backend(gm, example):
        box.append(ChoreoJITCompiler().compile_graph(gm, example))
        return lambda *a: tuple(torch.empty(s, dtype=d) for s, d in zip(box[0].launches[-1].out_shapes, box[0].launches[-1].out_dtypes))

    torch.compile(fn, backend=backend)(*args)
    return box[0]


def cache(B=2, Hq=4, Hkv=2, Sq=3, Skv=9, D=64):
    return torch.randn(B, Hq, Sq, D).bfloat16(), torch.randn(B, Hkv, Skv, D).bfloat16(), torch.randn(B, Hkv, Skv, D).bfloat16()


def test_the_definition_agrees_with_a_loop():
    """The tests' 64-bit reference against single rows written out."""
    q, k, v = cache(Sq=4, Skv=7)
    n = torch.tensor([2, 7])
    out, _ = reference(q, k, v, window=3, sinks=1, lengths=n)
    for b in range(2):
        for h in range(4):
            for i in range(4):
                p = int(n[b]) - 4 + i
                js = [j for j in range(int(n[b])) if j <= p and (j > p - 3 or j < 1)]
                want = torch.zeros(64, dtype=torch.float64)
                if js:
                    s = torch.stack([(q[b, h, i].double() @ k[b, h // 2, j].double()) / 8 for j in js])
                    want = torch.softmax(s, 0) @ torch.stack([v[b, h // 2, j].double() for j in js])
                assert torch.allclose(out[b, h, i], want, atol=1e-12)


def test_plans():
    q, k, v = cache()
    plan = compile_plan(lambda q, k, v, n: conductor.ops.window_attention(q, k, v, 5, 2, lengths=n), q, k, v, torch.tensor([3, 9]))
    (launch,) = plan.launches
    assert launch.template == Template.WINDOW_ATTENTION and len(launch.inputs) == 4 and launch.per_call_workspace
    assert (launch.params.window, launch.params.sinks, launch.params.has_lengths, launch.params.scale) == (5, 2, 1, 0.125)
    plan = compile_plan(lambda q, k, v: conductor.ops.prefix_attention(q, k[0], v[0], k, v, scale=0.5), q, k, v)
    assert plan.launches[-1].template == Template.PREFIX_ATTENTION and len(plan.launches[-1].inputs) == 5
    assert (plan.launches[-1].params.has_lengths, plan.launches[-1].params.scale) == (0, 0.5)
    plan = compile_plan(lambda q, k: torch.ops.conductor.window_attention(q, k, k, window=7), q, k)
    assert [b.name for b in plan.launches[0].inputs] == ["l_q_", "l_k_", "l_k_"] and plan.launches[0].params.window == 7


def test_only_the_batch_operands_are_sharded():
    q, k, v = cache(B=2, Hkv=2)
    n = torch.tensor([3, 9])
    dag = compile_plan(lambda q, k, v, n: conductor.ops.window_attention(q, k, v, 5, lengths=n), q, k, v, n).dag
    assert batch_inputs(dag) == (2, [0, 1, 2, 3])
    # the prefix has as many heads as the batch has sequences, and stays whole all the same
    dag = compile_plan(lambda q, a, b, k, v, n: conductor.ops.prefix_attention(q, a, b, k, v, lengths=n), q, k[0], v[0], k, v, n).dag
    assert batch_inputs(dag) == (2, [0, 3, 4, 5])
    dag = compile_plan(lambda q, a, k, n: torch.ops.conductor.prefix_attention(q, prefix_k=a, prefix_v=a, k=k, v=k, lengths=n), q, k[0], k, n).dag
    assert batch_inputs(dag) == (2, [0, 2, 3])


def test_refusals_before_any_launch():
    q, k, v = cache()
    with pytest.raises(DeviceError):
        conductor.ops.window_attention(q, k, v, 5)
    with pytest.raises(DeviceError):
        conductor.ops.prefix_attention(q, k[0], v[0], k, v)
    for shape, window, sinks in (((2, 4, 3, 64), 0, 0), ((2, 4, 3, 64), 3, -1), ((2, 4, 3, 96), 3, 0), ((4, 3, 64), 3, 0)):
        with pytest.raises(UnsupportedOperationError):
            kt.window_attention_launch("w", shape, torch.bfloat16, window, sinks, False, None)
    with pytest.raises(TypeError):
        kt.window_attention_launch("w", (2, 4, 3, 64), torch.bfloat16, 2.5, 0, False, None)
    with pytest.raises(UnsupportedOperationError):
        kt.prefix_attention_launch("p", (2, 4, 3, 80), torch.bfloat16, False, None)
    with pytest.raises((ConductorError, Exception)):
        compile_plan(lambda q, k, v: conductor.ops.window_attention(q, k, v, 0), q, k, v)


def _workspace(template, ins, out, params):
    lib = loader.load_library()
    n = ctypes.c_size_t(0)
    rc = lib.cdr_workspace_bytes(template, make_descriptors(ins), len(ins), make_descriptors([out]), 1,
                                 ctypes.cast(ctypes.byref(params), ctypes.c_void_p), ctypes.sizeof(params), ctypes.byref(n))
    return rc, lib.cdr_last_error().decode()


def test_arguments_are_checked_by_the_library(built_library):
    q, k, v = cache()
    n = torch.tensor([3, 9], dtype=torch.int32)

    def window(q=q, k=k, v=v, out=None, n=None, window=4, sinks=0, scale=0.1):
        ins = [q, k, v] + ([n] if n is not None else [])
        return _workspace(Template.WINDOW_ATTENTION, ins, torch.empty_like(q) if out is None else out,
                          kt.CdrWindowAttnParams(scale, 0 if n is None else 1, window, sinks))

    assert window()[0] == 0 and window(n=n)[0] == 0 and window(n=n.long())[0] == 0
    for bad, status, words in ((dict(window=0), -1, "window"), (dict(sinks=-1), -1, "sinks"), (dict(scale=0.0), -2, "scale"),
                               (dict(scale=float("inf")), -2, "scale"), (dict(q=q.float(), out=q.float()), -2, "dtype"),
                               (dict(k=k.half()), -1, "dtype"), (dict(k=k[:1], v=v[:1]), -1, "sequences"), (dict(v=v[:, :, :4]), -1, "same shapes"),
                               (dict(q=q[:, :3]), -1, "share"), (dict(n=n[:1]), -1, "lengths"), (dict(n=n.float()), -1, "lengths"),
                               (dict(q=q[0], out=q[0]), -1, "rank"), (dict(out=q[:1]), -1, "same shapes"),
                               (dict(k=k.transpose(2, 3).contiguous().transpose(2, 3)), -2, "contiguous"),
                               (dict(k=k[:, :, :1].expand(-1, -1, 9, -1)), -2, "stride"),
                               (dict(q=q.reshape(-1)[4:4 + 2 * 4 * 2 * 64].view(2, 4, 2, 64)), -3, "aligned"),
                               (dict(q=q[..., :32], k=k[..., :32], v=v[..., :32]), -2, "head dim")):
        rc, msg = window(**bad)
        assert rc == status and words in msg, (bad.keys(), rc, msg)

    def prefix(a, b):
        return _workspace(Template.PREFIX_ATTENTION, [q, a, b, k, v], torch.empty_like(q), kt.CdrPrefixAttnParams(0.1, 0))

    assert prefix(k[0], v[0])[0] == 0 and prefix(k[0, :, :0], v[0, :, :0])[0] == 0
    for a, b in ((k[0, :1], v[0, :1]), (k[0], v[0, :, :4]), (k[:1], v[:1]), (k[0].half(), v[0].half())):
        assert prefix(a, b)[0] == -1


def test_call_module_takes_only_the_tensors_it_was_made_for(built_library):
    """The compiled side of direct calls: anything else than the tensors of the first call is left to the caller."""
    from conductor.compiler.loader import load_call_module
    from conductor_b200.csrc.build import build_call_module

    build_call_module()
    module = load_call_module()
    item, ins, out = kt.CdrLaunchItem(), (kt.CdrTensor * 3)(), (kt.CdrTensor * 1)()
    q, k, v = cache()
    call = module.Call(ctypes.addressof(item), ctypes.addressof(ins), ctypes.addressof(out), 0, (q, k, v))
    shifted = torch.zeros(q.numel() + 1, dtype=q.dtype)[1:].view(q.shape)
    for bad in ((q, k), (q, k, v, v), (q, k, v[:1]), (q.half(), k, v), (q, k, v.transpose(1, 2).contiguous().transpose(1, 2)),
                (shifted, k, v), (q.clone().requires_grad_(), k, v), (q, k, None)):
        assert call.run(*bad) is None
    with pytest.raises(TypeError):
        module.Call(1, 2, 3, 4, (1, 2))
    with pytest.raises(TypeError):
        module.Call(1, 2)


def test_views_the_kernels_read_in_place():
    base = torch.zeros(2, 9, 4, 64, dtype=torch.bfloat16)
    assert attention_view_ok(base) and attention_view_ok(base.transpose(1, 2)) and attention_view_ok(base[:, 3:7, 1:2])
    assert not attention_view_ok(base.transpose(2, 3)) and not attention_view_ok(base[:1].expand(2, -1, -1, -1))
    assert not attention_view_ok(torch.zeros(2, 9, 4, 67, dtype=torch.bfloat16)[..., :64])
    assert not attention_view_ok(torch.zeros(2 * 64 + 1, dtype=torch.bfloat16)[1:].view(1, 1, 2, 64))
    assert attention_view_ok(torch.zeros(5, dtype=torch.int32)) and not attention_view_ok(torch.zeros(10, dtype=torch.int32)[::2])
