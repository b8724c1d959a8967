"""Callers and call forms of window_attention and prefix_attention that need no GPU: tracers, transforms, the call module."""
import ctypes
import json
import types

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

import conductor
from conductor.compiler import loader
from conductor.compiler.jit_compiler import ChoreoJITCompiler
from conductor.compiler.loader import load_call_module
from conductor.utils.exceptions import DeviceError, ExecutionError
from conductor_b200.codegen import kernel_templates as kt
from conductor_b200.csrc import build
from conductor_b200.csrc.build import CSRC, build_call_module
from conductor_b200.codegen.operator_registry import Template
from conductor_b200.utils.artifacts import DebugArtifactManager
from test_cache_attention import _workspace, cache, compile_plan

WINDOW, PREFIX = conductor.ops.window_attention, conductor.ops.prefix_attention


def test_symbolic_tracing_and_fake_tensors():
    def both(q, k, v, w, n):
        return WINDOW(q, k, v, w, 2, lengths=n) + PREFIX(q, k[0], v[0], k, v, lengths=n)

    names = [str(node.target) for node in torch.fx.symbolic_trace(both).graph.nodes if node.op == "call_function"]
    assert any("window_attention" in n for n in names) and any("prefix_attention" in n for n in names)
    q, k, v = cache()
    for device in ("cpu", "cuda"):
        with FakeTensorMode():
            args = [torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v)]
            out = both(*args, 4, torch.zeros(2, dtype=torch.int32, device=device))
        assert out.shape == q.shape and out.dtype == q.dtype and out.device.type == device


def test_the_dispatched_form_refuses_gradients():
    q, k, v = cache()
    window, prefix = torch.ops.conductor.window_attention, torch.ops.conductor.prefix_attention
    for call in (lambda: window(q.clone().requires_grad_(), k, v, 3), lambda: prefix(q, k[0].clone().requires_grad_(), v[0], k, v),
                 lambda: torch.func.grad(lambda q: window(q, k, v, 3).float().sum())(q),
                 lambda: torch.func.grad(lambda v: prefix(q, k[0], v[0], k, v=v).float().sum())(v)):
        with pytest.raises(ExecutionError, match="no backward"):
            call()
    with pytest.raises(ExecutionError, match="forward-mode"):
        torch.func.jvp(lambda q: window(q, k, v, 3), (q,), (torch.ones_like(q),))
    with fwAD.dual_level(), pytest.raises(ExecutionError, match="forward-mode"):
        prefix(fwAD.make_dual(q, q), k[0], v[0], k, v)


def test_call_module_leaves_to_the_dispatcher_what_is_its(built_library):
    """Tangents, dispatch modes, tracers and wrapped tensors: the kept call does not take them."""
    build_call_module()
    module = load_call_module()
    item, ins, out = kt.CdrLaunchItem(), (kt.CdrTensor * 3)(), (kt.CdrTensor * 1)()
    q, k, v = cache()
    call = module.Call(ctypes.addressof(item), ctypes.addressof(ins), ctypes.addressof(out), 0, (q, k, v))
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    def look(q, k, v):
        seen.append((call.run(q, k, v), module.is_dispatched(q, k, v)))
        return q

    assert not module.is_dispatched(q, k, v)
    with Mode():
        look(q, k, v)
    torch.jit.trace(look, (q, k, v), check_trace=False)
    torch.func.vmap(look)(*(t[None] for t in (q, k, v)))
    torch.func.functionalize(look)(q, k, v)
    assert seen == [(None, True)] * 4
    with fwAD.dual_level():
        assert call.run(q, fwAD.make_dual(k, k), v) is None


def test_strides_of_empty_operands_do_not_matter(built_library):
    q = cache()[0]
    for t in (torch.zeros(2, 2, 9, 67, dtype=q.dtype)[..., :64][:, :, :0], torch.zeros(2, 2, 64, 9, dtype=q.dtype).transpose(2, 3)[:, :, :0]):
        assert _workspace(Template.WINDOW_ATTENTION, [q, t, t], torch.empty_like(q), kt.CdrWindowAttnParams(0.1, 0, 4, 0))[0] == 0
        assert _workspace(Template.PREFIX_ATTENTION, [q, t[0], t[0], t, t], torch.empty_like(q), kt.CdrPrefixAttnParams(0.1, 0))[0] == 0


def test_every_launch_obeys_the_switch_that_puts_kernels_one_after_the_other():
    sources = [(f.name, line) for f in sorted(CSRC.glob("*.cu*")) for line in f.read_text().splitlines()]
    allowed = [(name, line) for name, line in sources if "programmaticStreamSerializationAllowed" in line]
    assert {name for name, _ in allowed} >= {"cdr_cache_attention.cu", "cdr_tile_attention.cu", "cdr_gemm.cu", "cdr_reduce.cu"}
    for name, line in allowed:
        assert "pdl_enabled()" in line, (name, line)
    assert sum("CDR_DISABLE_PDL" in line and "getenv" in line for _, line in sources) == 1


def test_window_and_sinks_may_change_from_call_to_call_of_a_compiled_function():
    torch._dynamo.reset()
    q, k, v = cache()
    seen = []

    def backend(gm, example):
        p = ChoreoJITCompiler().compile_graph(gm, example).launches[-1].params
        seen.append((p.window, p.sinks))
        return lambda *a: (torch.empty_like(q),)

    f = torch.compile(lambda q, k, v, w, s: conductor.ops.window_attention(q, k, v, w, s), backend=backend)
    numbers = [(5, 1), (6, 2), (7, 0), (70, 30)]
    for w, s in numbers:
        f(q, k, v, w, s)
    assert seen == numbers


def test_call_module_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    """A module of another torch or Python is built again however new its file is, and is not loaded."""
    ran = []
    monkeypatch.setattr(build, "CALL_MODULE_PATH", tmp_path / "_cdr_torch.so")
    monkeypatch.setattr(build, "CALL_MODULE_STAMP", tmp_path / "_cdr_torch.stamp")
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: ran.append(cmd) or types.SimpleNamespace(returncode=0, stdout="", stderr=""))
    build.CALL_MODULE_PATH.write_bytes(b"")
    build.CALL_MODULE_STAMP.write_text("torch 1.0 cpython-30")
    build.build_call_module()
    assert len(ran) == 1 and build.CALL_MODULE_STAMP.read_text() == build.call_module_identity()
    build.build_call_module()
    assert len(ran) == 1


def test_call_module_of_another_torch_is_not_loaded(built_library, monkeypatch):
    build_call_module()
    monkeypatch.setattr(loader, "_call_module", None)
    assert loader.load_call_module().built_for == build.call_module_identity()
    monkeypatch.setattr(loader, "_call_module", None)
    monkeypatch.setattr(build, "call_module_identity", lambda: "torch 1.0 cpython-30")
    with pytest.raises(DeviceError, match="was built for"):
        loader.load_call_module()


def test_the_library_is_built_without_the_call_module(monkeypatch):
    def fails(force=False):
        raise FileNotFoundError("g++")

    monkeypatch.setattr(build, "build_call_module", fails)
    monkeypatch.setattr(build, "build_library", lambda force=False, verbose=False: build.LIB_PATH)
    with pytest.warns(RuntimeWarning, match="call module"):
        assert build.build() == build.LIB_PATH


def test_a_compiled_call_with_a_window_of_nothing_is_refused():
    q, k, v = cache()
    for window, sinks in ((0, 0), (3, -1)):
        with pytest.raises(Exception, match="window must be at least 1 and sinks at least 0"):
            compile_plan(lambda q, k, v: conductor.ops.window_attention(q, k, v, window, sinks), q, k, v)


def test_debug_artifacts_name_the_operators(tmp_path):
    q, k, v = cache()
    plan = compile_plan(lambda q, k, v: conductor.ops.prefix_attention(conductor.ops.window_attention(q, k, v, 5), k[0], v[0], k, v), q, k, v)
    path = DebugArtifactManager(str(tmp_path)).save_clusters("kernel", plan.launches)
    names = [row["template"] for row in json.loads(path.read_text())]
    assert "window_attention" in names and "prefix_attention" in names and not any(n.isdigit() for n in names)


def test_scale_must_be_finite_in_powers_of_two(built_library):
    q, k, v = cache()
    for scale, status in ((2.3e38, 0), (2.4e38, -2), (float("nan"), -2), (1e-45, 0)):
        assert _workspace(Template.WINDOW_ATTENTION, [q, k, v], torch.empty_like(q), kt.CdrWindowAttnParams(scale, 0, 4, 0))[0] == status
        assert _workspace(Template.PREFIX_ATTENTION, [q, k[0], v[0], k, v], torch.empty_like(q), kt.CdrPrefixAttnParams(scale, 0))[0] == status
