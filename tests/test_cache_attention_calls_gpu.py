"""How window_attention and prefix_attention may be called: threads, transforms and tracers, views, single queries, repeats."""
import math
import os
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import conductor
from abi_util import execute_host
from cache_attention_ref import check, reference
from conductor.utils.exceptions import ExecutionError
from conductor_b200.compiler.gcu_backend import get_gcu_backend
from conductor_b200.codegen.kernel_templates import CdrWindowAttnParams
from conductor_b200.codegen.operator_registry import Template
from test_cache_attention_gpu import DEV, PREFIX, WINDOW, cache, lens, no_wait_gave_up, rand  # noqa: F401

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def in_a_new_thread(fn):
    """fn's result from a host thread that has made no CUDA call before; what it raises is raised here."""
    box = []

    def work():
        try:
            box.append((fn(), None))
        except BaseException as exc:  # noqa: BLE001 -- handed to the caller
            box.append((None, exc))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    out, exc = box[0]
    if exc is not None:
        raise exc
    return out


def test_calls_from_a_thread_without_a_context():
    """A new host thread has no CUDA context bound to it; everything it needs may be cached by then, so that no
    runtime call binds one before the library asks the driver for a tensor map or launches a run-time instance."""
    q, k, v = cache(4, 8, 2, 1, 600, 128)
    qp, kp, vp = cache(2, 4, 4, 300, 300, 128)
    pre = [rand(2, 3000, 128, seed=50 + i) for i in range(2)]
    x, w, b = rand(300, 256), rand(512, 256, seed=1), rand(512, seed=2)
    torch._dynamo.reset()
    get_gcu_backend().clear_cache()
    plans = []
    for fn, args in ((lambda x, w, b: torch.relu(torch.nn.functional.linear(x, w, b)), (x, w, b)),
                     (lambda q, k, v: torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True), (qp, kp, vp)),
                     (lambda x: torch.relu(x * 1.25 - 0.5) * torch.sigmoid(x) + 3.0 * x, (x,))):      # a run-time instance
        torch.compile(fn, backend="gcu")(*args)
        plans.append((list(get_gcu_backend()._compiled_functions.values())[-1], args))
    calls = [lambda: WINDOW(q, k, v, 256, 4), lambda: WINDOW(qp, kp, vp, 100, 4), lambda: PREFIX(q, *pre, k, v)]
    calls += [lambda p=p, a=a: p(*a)[0] for p, a in plans]
    for call in calls:
        want = call().clone()
        call()                                   # leaves a free block of every size the call takes
        torch.cuda.synchronize()
        for _ in range(2):
            assert torch.equal(in_a_new_thread(call), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,P,D", [(13, 14, 2, 3, 5003, 64), (40, 14, 2, 3, 3000, 128), (5, 32, 8, 1, 16000, 128)])
def test_packed_rows_do_not_depend_on_what_ran_before(B, Hq, Hkv, Sq, P, D, dtype):
    """The rows of the packed product that no query fills: the same bits whatever earlier kernels left in shared memory."""
    q, k, v = cache(B, Hq, Hkv, Sq, 40, D, dtype=dtype, seed=B)
    pre = [rand(Hkv, P, D, dtype=dtype, seed=50 + i) for i in range(2)]
    full = cache(64, 8, 2, 4, 40, D, dtype=dtype, seed=3)           # 16 rows per sequence: all 128 rows in use
    long = [rand(2, 20000, D, dtype=dtype, seed=60 + i) for i in range(2)]
    first = None
    for size in (0.0, 1.0, 30.0, 100.0, 0.0, 300.0):
        PREFIX(full[0] * size, *long, *full[1:])
        got = PREFIX(q, *pre, k, v)
        first = got if first is None else first
        assert torch.equal(got, first), size
    check(first, reference(q, k, v, prefix=pre))


@pytest.mark.parametrize("B,Hq,Hkv,Skv,D,window,sinks", [(64, 8, 8, 2000, 128, 16, 1000), (32, 32, 8, 4500, 128, 128, 4096), (150, 8, 8, 700, 64, 1, 333)])
def test_hidden_keys_of_a_single_query_with_many_sinks(B, Hq, Hkv, Skv, D, window, sinks):
    """With one query per sequence hidden keys may hold anything, however many sequences and sinks there are."""
    q, k, v = cache(B, Hq, Hkv, 1, Skv, D)
    want = WINDOW(q, k, v, window, sinks)
    few = slice(0, 3)
    check(want[few], reference(q[few], k[few], v[few], window=window, sinks=sinks))
    k[:, :, sinks:Skv - window], v[:, :, sinks:Skv - window] = float("nan"), float("inf")
    assert torch.equal(WINDOW(q, k, v, window, sinks), want)


def test_forward_mode_is_refused():
    q, k, v = cache(2, 4, 2, 3, 50, 64)
    pre = [rand(2, 30, 64, seed=50 + i) for i in range(2)]
    WINDOW(q, k, v, 20), PREFIX(q, *pre, k, v)                      # the kept form of both calls exists
    with fwAD.dual_level():
        d = fwAD.make_dual(q, torch.ones_like(q))
        for call in (lambda: WINDOW(d, k, v, 20), lambda: torch.ops.conductor.window_attention(d, k, v, 20),
                     lambda: PREFIX(d, *pre, k, v), lambda: PREFIX(q, fwAD.make_dual(pre[0], pre[1]), pre[1], k, v)):
            with pytest.raises(ExecutionError, match="forward-mode"):
                call()
        WINDOW(q, k, v, 20)                                         # no tangent: as ever
        with fwAD._set_fwd_grad_enabled(False):
            WINDOW(d, k, v, 20)


def test_function_transforms_are_refused():
    q, k, v = cache(2, 4, 2, 3, 50, 64)
    f = lambda q: WINDOW(q, k, v, 20).float().sum()                 # noqa: E731
    for call in (lambda: torch.func.grad(f)(q), lambda: torch.func.jvp(f, (q,), (torch.ones_like(q),)),
                 lambda: torch.func.vjp(f, q), lambda: torch.ops.conductor.window_attention(q.clone().requires_grad_(), k, v, 20)):
        with pytest.raises(ExecutionError, match="backward|forward-mode"):
            call()


def test_tracers_record_the_operators():
    """What a tracer returns computes the operator on other inputs, not the memory that the traced call filled."""
    from torch.fx.experimental.proxy_tensor import make_fx

    q, k, v = cache(2, 4, 2, 3, 50, 64)
    pre = [rand(2, 30, 64, seed=50 + i) for i in range(2)]
    n = lens(50, 31)
    both = lambda q, k, v, a, b: WINDOW(q, k, v, 20, 2, lengths=n) + PREFIX(q, a, b, k, v, lengths=n)      # noqa: E731
    other = [t.flip(0).contiguous() for t in (q, k, v)] + [t.flip(1).contiguous() for t in pre]
    want = both(*other)
    g = make_fx(both)(q, k, v, *pre)
    names = [str(node.target) for node in g.graph.nodes if node.op == "call_function"]
    assert "conductor.window_attention.default" in names and "conductor.prefix_attention.default" in names
    assert torch.equal(g(*other), want)
    traced = torch.jit.trace(both, (q, k, v, *pre))
    assert "conductor::window_attention" in str(traced.inlined_graph)
    assert torch.equal(traced(*other), want)
    assert torch.equal(both(*other), want)


def test_views_of_empty_tensors():
    """An empty cache or prefix has no element to read: its strides do not matter."""
    q = rand(2, 4, 3, 64)
    odd = rand(2, 2, 9, 67)[..., :64][:, :, :0]
    turned = rand(2, 2, 64, 9).transpose(2, 3)[:, :, :0]
    for t in (odd, turned):
        assert torch.equal(WINDOW(q, t, t, 5), torch.zeros_like(q))
        k, v = rand(2, 2, 50, 64, seed=1), rand(2, 2, 50, 64, seed=2)
        assert torch.equal(PREFIX(q, t[0], t[0], k, v), WINDOW(q, k, v, 1 << 20))


def test_views_inside_and_into_compiled_functions():
    """Token-major caches, slices and a fused projection: as graph inputs (read in place) and made in the graph (gathered)."""
    B, Hq, Hkv, Sq, Skv, D = 3, 8, 2, 5, 120, 64
    q, k, v = cache(B, Hq, Hkv, Sq, Skv, D)
    n = lens(120, 77, 4)
    want = reference(q, k, v, window=40, sinks=3, lengths=n)
    turned = [t.transpose(1, 2).contiguous() for t in (q, k, v)]
    torch._dynamo.reset()
    outside = torch.compile(lambda q, k, v, n: conductor.ops.window_attention(q, k, v, 40, 3, lengths=n), backend="gcu")
    check(outside(*(t.transpose(1, 2) for t in turned), n), want, "views as inputs")
    inside = torch.compile(lambda q, k, v, n: conductor.ops.window_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), 40, 3, lengths=n),
                           backend="gcu")
    check(inside(*turned, n), want, "views in the graph")
    longer = [torch.cat([t, t.flip(2)], 2) for t in (k, v)]
    sliced = torch.compile(lambda q, k, v, n: conductor.ops.window_attention(q, k[:, :, :Skv], v[:, :, :Skv], 40, 3, lengths=n), backend="gcu")
    check(sliced(q, *longer, n), want, "slices in the graph")


def test_numbers_of_a_compiled_function_change():
    """Window and sinks are plain numbers of the call: other values are another plan, not a refusal."""
    q, k, v = cache(2, 4, 2, 3, 90, 64)
    torch._dynamo.reset()
    f = torch.compile(lambda q, k, v, w, s: conductor.ops.window_attention(q, k, v, w, s), backend="gcu")
    for w, s in ((5, 1), (6, 2), (70, 30), (7, 3)):
        check(f(q, k, v, w, s), reference(q, k, v, window=w, sinks=s), f"{w} {s}")


def test_the_same_bits_with_kernels_one_after_the_other(tmp_path):
    """CDR_DISABLE_PDL=1: no kernel starts before the one in front of it has ended; the results are the same."""
    code = """
import sys
sys.path[:0] = [%r, %r]
import torch
from test_cache_attention_gpu import PREFIX, WINDOW, cache, lens, rand
q, k, v = cache(20, 8, 2, 1, 600, 128)
n = torch.arange(20, device="cuda", dtype=torch.int32) * 30
pre = [rand(2, 3000, 128, seed=50 + i) for i in range(2)]
few = [t[:2].contiguous() for t in (q, k, v)]
long = cache(20, 8, 2, 300, 300, 64)
out = []
for _ in range(3):
    out += [WINDOW(q, k, v, 256, 4, lengths=n), PREFIX(q, *pre, k, v, lengths=n), WINDOW(*few, 100), PREFIX(*few[:1], *pre, *few[1:]), WINDOW(*long, 100, 4)]
torch.save([t.cpu() for t in out], sys.argv[1])
""" % (str(ROOT), str(ROOT / "tests"))
    got = []
    for i, extra in enumerate(({}, {"CDR_DISABLE_PDL": "1"})):
        path = tmp_path / f"{i}.pt"
        subprocess.run([sys.executable, "-c", code, str(path)], env={**os.environ, **extra}, check=True, timeout=300)
        got.append(torch.load(path))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("B,H,Sq,keys,P", [(1, 1, 1, 100000, 0), (1, 2, 3, 9000, 0), (40, 2, 1, 20000, 0), (2, 1, 300, 16000, 0), (40, 2, 1, 64, 16000)])
def test_small_f16_weights_beside_a_dominating_key(B, H, Sq, keys, P):
    """One key of weight 1 with value 0 and many of weight 2^-25.6, below what f16 holds, with value 1.

    Scores are exact.  A weight w counts to within 2^-32 of the largest (half a step of the smallest f16, seven binary places down), the
    output is rounded once (2^-11 relative, 2^-25 below the smallest normal); fp32 sums and exponentials: 2^-18."""
    def near(*shape):
        k = torch.zeros(*shape, 64, dtype=torch.float16, device=DEV)
        v = torch.ones_like(k)
        k[..., 0, 0], v[..., 0, :] = 17.75, 0.0
        return k, v

    q = torch.zeros(B, H, Sq, 64, dtype=torch.float16, device=DEV)
    q[..., 0] = 8.0                                                 # score = the key's first element
    weight = math.exp(-17.75)
    if P:
        k = torch.zeros(B, H, keys, 64, dtype=torch.float16, device=DEV)
        got = PREFIX(q, *near(H, P), k, torch.ones_like(k))
    else:
        got = WINDOW(q, *near(B, H, keys), 1 << 30)
    seen = torch.arange(keys - Sq, keys, device=DEV, dtype=torch.float64) + P      # keys of weight 2^-25.6 that row i sees
    want = (seen * weight / (1 + seen * weight)).view(1, 1, Sq, 1)
    bound = seen.view(1, 1, Sq, 1) * 2.0 ** -32 + want * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -25
    assert ((got.double() - want).abs() <= bound).all(), (got.flatten()[0].item(), want.flatten()[0].item())


def test_host_tensors_of_any_alignment():
    """The host entry point stages its tensors: where they lie in host memory does not matter."""
    q, k, v = cache(2, 4, 2, 3, 90, 64)
    p = CdrWindowAttnParams(0.125, 0, 20, 2)
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    out = torch.empty(q.numel() + 1, dtype=q.dtype)[1:].view(q.shape)
    assert all(t.data_ptr() % 16 for t in (*odd, out))
    assert execute_host(Template.WINDOW_ATTENTION, odd, [out], p) == 0
    check(out.to(DEV), reference(q, k, v, window=20, sinks=2))
