"""window_attention and prefix_attention on a GPU against their definition in 64 bits."""
import ctypes
import threading

import pytest
import torch

import conductor
from abi_util import execute_host, launch, workspace_bytes
from cache_attention_ref import check, reference
from conductor.compiler.loader import load_library
from conductor_b200.codegen.kernel_templates import CdrWindowAttnParams
from conductor_b200.codegen.operator_registry import Template
from conductor.utils.exceptions import DeviceError, ExecutionError, UnsupportedOperationError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WINDOW, PREFIX = conductor.ops.window_attention, conductor.ops.prefix_attention


def rand(*shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def cache(B, Hq, Hkv, Sq, Skv, D, dtype=torch.bfloat16, seed=0):
    return rand(B, Hq, Sq, D, dtype=dtype, seed=seed), rand(B, Hkv, Skv, D, dtype=dtype, seed=seed + 1), rand(B, Hkv, Skv, D, dtype=dtype, seed=seed + 2)


def lens(*n, dtype=torch.int32):
    return torch.tensor(n, dtype=dtype, device=DEV)


@pytest.fixture(autouse=True, scope="module")
def no_wait_gave_up():
    """Every device-side wait of these tests ended by its signal, not by its limit."""
    yield
    word = ctypes.c_int(0)
    assert load_library().cdr_device_status(ctypes.byref(word), 1) == 0, hex(word.value)


SHAPES = [
    # B, Hq, Hkv, Sq, Skv, D
    (1, 1, 1, 1, 1, 64), (2, 8, 2, 1, 300, 128), (3, 7, 1, 1, 1000, 64), (1, 32, 8, 1, 4097, 128),
    (2, 4, 4, 5, 77, 64), (1, 6, 2, 17, 130, 128), (2, 3, 3, 33, 33, 64), (1, 2, 1, 129, 257, 128),
    (1, 4, 2, 300, 300, 64), (2, 2, 2, 511, 640, 128), (1, 5, 1, 260, 1025, 64), (1, 2, 2, 1030, 1030, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 1), (100, 4), (128, 128), (333, 300), (1 << 40, 0)])
def test_window_matches_the_definition(shape, dtype, window, sinks):
    q, k, v = cache(*shape, dtype=dtype, seed=sum(shape))
    check(WINDOW(q, k, v, window, sinks), reference(q, k, v, window=window, sinks=sinks), f"{shape} {window} {sinks}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("P", [0, 1, 15, 128, 777])
def test_prefix_matches_the_definition(shape, dtype, P):
    q, k, v = cache(*shape, dtype=dtype, seed=sum(shape))
    pre = [rand(shape[2], P, shape[5], dtype=dtype, seed=50 + i) for i in range(2)]
    check(PREFIX(q, *pre, k, v), reference(q, k, v, prefix=pre), f"{shape} {P}")


@pytest.mark.parametrize("Hq,Hkv,Sq,Skv", [(8, 2, 1, 200), (4, 4, 3, 200), (2, 1, 40, 200), (2, 2, 200, 200), (3, 1, 300, 700), (24, 1, 1, 500)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_lengths(Hq, Hkv, Sq, Skv, index):
    """Ragged lengths, none, one, more than the cache and negative ones; NaN and infinities behind them."""
    n = [0, 1, 2, Sq - 1, Sq, Sq + 1, 127, 128, 129, Skv - 1, Skv, Skv + 5, -3]
    lengths = lens(*n, dtype=index)
    q, k, v = cache(len(n), Hq, Hkv, Sq, Skv, 64, seed=7)
    for b, m in enumerate(n):
        for t, junk in ((k, float("nan")), (v, float("inf"))):
            t[b, :, min(max(m, 0), Skv):] = junk
    pre = [rand(Hkv, 150, 64, seed=50 + i) for i in range(2)]
    for window, sinks in ((50, 3), (1000, 0)):
        check(WINDOW(q, k, v, window, sinks, lengths=lengths), reference(q, k, v, window=window, sinks=sinks, lengths=lengths), f"{window}")
    check(PREFIX(q, *pre, k, v, lengths=lengths), reference(q, k, v, lengths=lengths, prefix=pre), "prefix")


@pytest.mark.parametrize("B,Hq,Hkv,Sq,P,D", [(2, 8, 8, 1, 900, 64), (20, 32, 8, 1, 600, 128), (130, 8, 1, 1, 1000, 64), (9, 14, 2, 3, 513, 128),
                                             (70, 4, 4, 5, 300, 64), (300, 2, 2, 1, 128, 128), (3, 16, 1, 8, 257, 64), (2, 16, 1, 9, 257, 64), (5, 200, 1, 1, 140, 128),
                                             (13, 14, 2, 3, 5003, 64), (33, 32, 4, 1, 3000, 128), (257, 8, 2, 1, 2000, 64)])
def test_prefix_of_many_sequences(B, Hq, Hkv, Sq, P, D):
    q, k, v = cache(B, Hq, Hkv, Sq, 40, D, seed=B)
    lengths = torch.arange(B, device=DEV) * 7 % 41
    pre = [rand(Hkv, P, D, seed=50 + i) for i in range(2)]
    check(PREFIX(q, *pre, k, v, lengths=lengths), reference(q, k, v, lengths=lengths, prefix=pre))


def test_hidden_keys_of_a_single_query_may_hold_anything():
    q, k, v = cache(2, 8, 2, 1, 400, 128)
    want = reference(q, k, v, window=100, sinks=5)
    k[:, :, 5:300], v[:, :, 5:300] = float("nan"), float("inf")
    check(WINDOW(q, k, v, 100, 5), want)


@pytest.mark.parametrize("Sq,Skv", [(1, 500), (300, 500)])
def test_masked_scores_of_the_lowest_value_and_large_scores(Sq, Skv):
    """Scores of the size where a weight is 0 or 1, growing and falling along the keys (rescales)."""
    q, k, v = cache(1, 4, 2, Sq, Skv, 64)
    k = k * torch.linspace(0.01, 20, Skv, device=DEV).view(1, 1, -1, 1).to(k.dtype)
    for kk in (k, k.flip(2).contiguous()):
        check(WINDOW(q, kk, v, 200, 7), reference(q, kk, v, window=200, sinks=7))
        check(WINDOW(q, kk, v, 9999, 0, scale=0.9), reference(q, kk, v, window=9999, scale=0.9))


@pytest.mark.parametrize("Sq", [1, 3, 200, 300])
def test_views_are_read_in_place(Sq):
    B, Hq, Hkv, Skv, D = 2, 8, 2, 333, 64
    q, k, v = cache(B, Hq, Hkv, Sq, Skv, D)
    want = reference(q, k, v, window=77, sinks=4)
    token_major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    check(WINDOW(*token_major, 77, 4), want, "token-major")
    fused = torch.cat([t.transpose(1, 2).reshape(B, -1, t.shape[1] * D) for t in (k, v)], 2)      # one [B, S, 2*Hkv*D] projection
    kf, vf = (t.view(B, Skv, Hkv, D).transpose(1, 2) for t in fused.split(Hkv * D, 2))
    assert not kf.is_contiguous()
    check(WINDOW(q, kf, vf, 77, 4), want, "fused projection")
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    check(WINDOW(*odd, 77, 4), want, "misaligned")
    strided = [torch.empty(*t.shape[:-1], D + 3, dtype=t.dtype, device=DEV)[..., :D].copy_(t) for t in (q, k, v)]
    check(WINDOW(*strided, 77, 4), want, "odd pitch")
    one = rand(1, Hkv, Skv, D, seed=1).expand(B, -1, -1, -1)                                      # broadcast over the batch
    check(WINDOW(q, one, one, 77, 4), reference(q, one, one, window=77, sinks=4), "broadcast")
    pre = rand(300, Hkv, D, seed=9).transpose(0, 1)
    check(PREFIX(token_major[0], pre, pre, *token_major[1:]), reference(q, k, v, prefix=(pre, pre)), "prefix")


@pytest.mark.parametrize("B,Sq,Skv,P", [(1, 1, 3000, 0), (70, 1, 900, 0), (2, 300, 500, 0), (40, 1, 200, 1500)])
def test_nan_in_a_query_stays_in_its_row(B, Sq, Skv, P):
    q, k, v = cache(B, 8, 2, Sq, Skv, 64)
    pre = [rand(2, P, 64, seed=50 + i) for i in range(2)]
    call = (lambda q: PREFIX(q, *pre, k, v)) if P else (lambda q: WINDOW(q, k, v, 1 << 20))
    clean = call(q)
    broken = q.clone()
    broken[B // 2, 3, Sq // 2, 5] = float("nan")
    got = call(broken)
    assert got[B // 2, 3, Sq // 2].isnan().all()
    got[B // 2, 3, Sq // 2] = clean[B // 2, 3, Sq // 2]
    assert torch.equal(got, clean)


def test_thousands_of_sequences():
    """More sequences than the table of units has entries; lengths as a strided view and behind an odd offset."""
    B = 5000
    q, k, v = cache(B, 2, 1, 1, 40, 64)
    n = (torch.arange(2 * B, device=DEV, dtype=torch.int32) * 7919) % 41
    every_other, shifted = n[::2], n[1:B + 1]
    assert not every_other.is_contiguous()
    for lengths in (every_other, shifted):
        got = WINDOW(q, k, v, 9, 2, lengths=lengths)
        scores = torch.einsum("bhqd,bkd->bhqk", q.double(), k[:, 0].double()) / 8
        key, last = torch.arange(40, device=DEV).view(1, 1, 1, 40), lengths.view(B, 1, 1, 1) - 1
        seen = (key <= last) & ((key > last - 9) | (key < 2))
        w = torch.softmax(scores.masked_fill(~seen, float("-inf")), -1).nan_to_num(0.0)
        want = torch.einsum("bhqk,bkd->bhqd", w, v[:, 0].double())
        bound = 2.0 ** -8 * (torch.einsum("bhqk,bkd->bhqd", w, v[:, 0].double().abs()) + want.abs()) * 1.02 + 1e-6
        assert ((got.double() - want).abs() <= bound).all()


def test_empty_calls():
    q, k, v = cache(2, 4, 2, 3, 0, 64)
    assert torch.equal(WINDOW(q, k, v, 5), torch.zeros_like(q))
    assert WINDOW(q[:0], k[:0], v[:0], 5).shape == (0, 4, 3, 64)
    assert WINDOW(q[:, :, :0], k, v, 5).shape == (2, 4, 0, 64)
    pre = rand(2, 10, 64)
    assert torch.equal(PREFIX(q, pre, pre, k, v), torch.zeros_like(q))       # no own keys: every query is padding
    q = rand(2, 4, 300, 64)
    assert torch.equal(WINDOW(q, k, v, 5), torch.zeros_like(q)) and torch.equal(PREFIX(q, pre, pre, k, v), torch.zeros_like(q))


def test_refusals():
    q, k, v = cache(2, 4, 2, 3, 9, 64)
    for bad in (lambda: WINDOW(q, k, v, 0), lambda: WINDOW(q, k, v, 4, -1), lambda: WINDOW(q.float(), k.float(), v.float(), 4),
                lambda: WINDOW(q[..., :32], k[..., :32], v[..., :32], 4), lambda: WINDOW(q, k, v, 4, scale=0.0),
                lambda: WINDOW(q, k, v, 4, scale=float("nan"))):
        with pytest.raises(UnsupportedOperationError):
            bad()
    for bad in (lambda: WINDOW(q, k[:1], v, 4), lambda: WINDOW(q, k, v[:, :1], 4), lambda: WINDOW(q[:, :3], k, v, 4),
                lambda: WINDOW(q, k.half(), v.half(), 4), lambda: WINDOW(q, k, v, 4, lengths=lens(1)),
                lambda: WINDOW(q, k, v, 4, lengths=lens(1, 2).float()), lambda: PREFIX(q, k, v, k, v),
                lambda: PREFIX(q, k[0, :1], v[0, :1], k, v), lambda: PREFIX(q, k[0], v[0, :, :3], k, v)):
        with pytest.raises(ExecutionError):
            bad()
    with pytest.raises(DeviceError):
        WINDOW(q.cpu(), k.cpu(), v.cpu(), 4)
    with pytest.raises(ExecutionError):
        WINDOW(q, k, v, 4, lengths=torch.tensor([1, 2]))
    with pytest.raises(ExecutionError, match="requires grad"):
        WINDOW(q.requires_grad_(), k, v, 4)
    with torch.no_grad():
        WINDOW(q, k, v, 4)


def test_long_cache_offsets_pass_32_bits():
    """A cache of more than 2^32 bytes per tensor, most of it untouched: the last sequence's keys lie beyond."""
    B, Hkv, Skv, D = 3, 8, 1 << 20, 128
    k = torch.empty(B, Hkv, Skv, D, dtype=torch.bfloat16, device=DEV)
    assert k.numel() * 2 > 1 << 32
    v = torch.empty_like(k)
    n = 700
    for t, s in ((k, 1), (v, 2)):
        t[:, :, -n:] = rand(B, Hkv, n, D, seed=s)
        t[:, :, :2] = rand(B, Hkv, 2, D, seed=s + 10)
    for Sq in (1, 130):
        q = rand(B, 16, Sq, D, seed=3)
        got = WINDOW(q, k, v, 500, 2)
        ks, vs = (torch.cat([t[:, :, :2], t[:, :, -n:]], 2) for t in (k, v))      # the same keys, packed
        check(got, reference(q, ks, vs, window=500, sinks=2), f"{Sq}")


def test_other_streams_and_graph_replay():
    q, k, v = cache(4, 8, 2, 1, 600, 128)
    pre = [rand(2, 800, 128, seed=50 + i) for i in range(2)]
    qp, kp, vp = cache(1, 4, 2, 300, 300, 64)

    def calls():
        return WINDOW(q, k, v, 256, 4), PREFIX(q, *pre, k, v), WINDOW(qp, kp, vp, 100, 4)

    want = [t.clone() for t in calls()]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(calls())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for ts in got for a, b in zip(ts, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = calls()
        graphs.append((g, outs))
    for _ in range(5):
        for s, (g, _o) in zip(streams, graphs):      # two captured graphs in flight at a time
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _g, outs in graphs:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    q.copy_(rand(*q.shape, seed=99))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], calls()))


def test_more_tiles_than_processors_in_a_graph():
    """Tiles are drawn from a counter in scratch: every replay starts it again, on each of two graphs at once."""
    q, k, v = cache(20, 8, 2, 300, 300, 64)
    n = torch.arange(20, device=DEV) * 17
    want = WINDOW(q, k, v, 100, 4, lengths=n)
    check(want, reference(q, k, v, window=100, sinks=4, lengths=n))
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = WINDOW(q, k, v, 100, 4, lengths=n)
        graphs.append((g, out))
    for _ in range(4):
        for s, (g, _o) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _g, out in graphs)


def test_calls_from_several_threads():
    q, k, v = cache(4, 8, 2, 1, 600, 128)
    want = WINDOW(q, k, v, 256, 4)
    bad = []

    def work(seed):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(50):
                if not torch.equal(WINDOW(q, k, v, 256, 4), want):
                    bad.append((seed, i))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_captured_sequence_with_runs_in_flight():
    """Runs of one plan on branches of one graph: each has its own scratch (tile counter, partial results)."""
    from conductor_b200.compiler.gcu_backend import get_gcu_backend

    torch._dynamo.reset()
    get_gcu_backend().clear_cache()
    sets = [tuple(cache(20, 8, 2, 300, 300, 64, seed=10 * i)) for i in range(4)]
    f = torch.compile(lambda q, k, v: conductor.ops.window_attention(q, k, v, 100, 4) * 2.0, backend="gcu")
    want = [f(*s).clone() for s in sets]
    plan = list(get_gcu_backend()._compiled_functions.values())[-1]
    seq = plan.capture_sequence(sets, lanes=2)
    for _ in range(3):
        seq.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o[0], w) for o, w in zip(seq.all_outputs, want))


def test_library_calls_with_strided_output_and_host_tensors():
    q, k, v = cache(2, 4, 2, 3, 90, 64)
    n = lens(90, 41)
    p = CdrWindowAttnParams(0.125, 1, 20, 2)
    want = reference(q, k, v, window=20, sinks=2, lengths=n)
    out = torch.full((2, 3, 4, 64 + 8), 7.0, dtype=q.dtype, device=DEV)
    view = out[..., :64].transpose(1, 2)
    ws = torch.empty(max(1, workspace_bytes(Template.WINDOW_ATTENTION, [q, k, v, n], [view], p)), dtype=torch.uint8, device=DEV)
    launch(Template.WINDOW_ATTENTION, [q, k, v, n], [view], p, workspace=ws)
    check(view, want)
    assert (out[..., 64:] == 7.0).all()                       # what lies between the rows is left as it was
    host = torch.empty(q.shape, dtype=q.dtype)
    assert execute_host(Template.WINDOW_ATTENTION, [t.cpu() for t in (q, k, v, n)], [host], p) == 0
    check(host.to(DEV), want)
    long_q = rand(40, 8, 300, 64)
    lk, lv = rand(40, 2, 300, 64, seed=1), rand(40, 2, 300, 64, seed=2)
    p = CdrWindowAttnParams(0.125, 0, 64, 0)
    assert launch(Template.WINDOW_ATTENTION, [long_q, lk, lv], [torch.empty_like(long_q)], p, check=False) == -6      # no workspace
    assert launch(Template.WINDOW_ATTENTION, [long_q, lk, lv], [torch.empty_like(long_q)], p,
                  workspace=torch.empty(4096, dtype=torch.uint8, device=DEV)[8:], check=False) == -3


def test_the_same_call_gives_the_same_bits():
    q, k, v = cache(3, 8, 2, 2, 999, 128)
    pre = [rand(2, 2000, 128, seed=50 + i) for i in range(2)]
    first = WINDOW(q, k, v, 500, 4), PREFIX(q, *pre, k, v)
    for _ in range(5):
        assert torch.equal(WINDOW(q, k, v, 500, 4), first[0]) and torch.equal(PREFIX(q, *pre, k, v), first[1])


def test_compiled_graphs_with_both_calling_conventions():
    torch._dynamo.reset()

    def block(q, k, v, pk, pv, n):
        o = conductor.ops.window_attention(q, k, v, 60, 4, lengths=n)
        return conductor.ops.prefix_attention(torch.relu(o), pk, pv, k, v, lengths=n) + q

    q, k, v = cache(3, 4, 2, 5, 200, 64)
    pre = [rand(2, 90, 64, seed=50 + i) for i in range(2)]
    n = lens(200, 100, 3)
    first = torch.relu(WINDOW(q, k, v, 60, 4, lengths=n))
    second, tol = reference(first, k, v, lengths=n, prefix=pre)
    want = (second + q.double(), tol + 2.0 ** -8 * ((second + q.double()).abs() + second.abs()) * 1.01)
    f = torch.compile(block, backend="gcu")
    check(f(q, k, v, *pre, n), want, "device")
    check(f(*(t.cpu() for t in (q, k, v, *pre, n))).to(DEV), want, "host")
    with pytest.raises(Exception, match="requires grad|no backward"):
        f(q.requires_grad_(), k, v, *pre, n)


def test_prompt_chunks_and_decode_steps_agree():
    """As a server uses them: a prompt in chunks, then tokens one by one, sequences of different lengths
    in one cache; and the same cache behind a shared prefix."""
    B, Hq, Hkv, S, D, W, sinks = 3, 8, 2, 400, 64, 96, 4
    q, k, v = cache(B, Hq, Hkv, S, S, D)
    whole = reference(q, k, v, window=W, sinks=sinks)
    used = torch.full_like(k, float("nan")), torch.full_like(v, float("nan"))
    done = 0
    for step in (150, 130, 37, 3, 1, 1, 1):
        for t, src in zip(used, (k, v)):
            t[:, :, done:done + step] = src[:, :, done:done + step]
        done += step
        n = lens(*[done] * B)
        got = WINDOW(q[:, :, done - step:done], *used, W, sinks, lengths=n)
        check(got, [t[:, :, done - step:done] for t in whole], f"step of {step}")
    # a prefix is the same attention over the joined keys
    pk, pv = k[0, :, :250], v[0, :, :250]
    own_k, own_v = k[:, :, 250:], v[:, :, 250:]
    for Sq in (1, 4, 150):
        joined = [torch.cat([p.expand(B, -1, -1, -1), o], 2) for p, o in ((pk, own_k), (pv, own_v))]
        got = PREFIX(q[:, :, -Sq:], pk, pv, own_k, own_v)
        check(got, reference(q[:, :, -Sq:], *joined, window=1 << 20), f"prefix, {Sq}")
        check(WINDOW(q[:, :, -Sq:], *joined, 1 << 20), reference(q[:, :, -Sq:], *joined, window=1 << 20), f"joined, {Sq}")
