"""The operators over rows of many classes where calls meet: captured into graphs that are replayed between eager work, on
streams and host threads of their own, in place on few long rows, and on arrays beyond 2^32 elements."""
import ctypes
import threading

import numpy as np
import pytest
import torch

import class_rows_ref as ref
from anode_amd import gpu
from anode_amd._lib import load
from gpu_util import F32, call, dev, host
from test_gpu_class_rows import check_distill, drafts, got_u32, logits, rounded, slots, u32

pytestmark = pytest.mark.gpu


class Chain:
    """All of the operators on shapes that need scratch and on shapes that do not: (classes, rows, k) each."""

    SHAPES = [(100003, 3, 20), (1000, 40, 5)]

    def __init__(self, seed):
        g = np.random.default_rng(seed)
        self.parts = []
        for n, rows, k in self.SHAPES:
            target, draft, token = drafts(g, n, 2, 2)
            self.parts.append({
                "n": n, "rows": rows, "k": k, "x": dev(logits(g, rows, n, "f32")),
                "teacher": dev(logits(g, rows, n, "bf16")).to(torch.bfloat16), "dy": dev(g.standard_normal(rows).astype(F32)),
                "target": dev(target), "draft": dev(draft), "token": u32(token), "accept": dev(g.random((2, 2)).astype(F32)),
                "pick": dev(g.random(2).astype(F32))})

    def outputs(self):
        out = []
        for p in self.parts:
            n, rows, k = p["n"], p["rows"], p["k"]
            f = lambda m: torch.full((m,), float("nan"), device="cuda")  # noqa: E731
            i = lambda m: torch.full((m,), 7, dtype=torch.int32, device="cuda")  # noqa: E731
            out.append({"value": f(rows * k), "index": i(rows * k), "norm": f(rows), "loss": f(rows), "top": f(rows), "total": f(rows),
                        "dx": f(rows * n), "loss2": f(rows), "top2": f(rows), "total2": f(rows), "dx2": f(rows * n),
                        "tokens": i(6), "accepted": i(2)})
        return out

    def run(self, outs, stream=None):
        for p, o in zip(self.parts, outs):
            n, rows, k = p["n"], p["rows"], p["k"]
            head = (n, rows, 0, k, 2.0)
            def go(name, *args):
                assert gpu.call(name, *args, stream=stream) == 0, name
            go("anode_gpu_top_k_rows_bf16", n, rows, 0, k, 2.0, p["teacher"], o["value"], o["index"], o["norm"])
            teacher = (o["value"], o["index"], o["norm"])
            go("anode_gpu_softmax_distill_fused_fwd_bwd_rows_f32", *head, p["x"], *teacher, p["dy"], o["loss"], o["top"], o["total"],
               o["dx"])
            go("anode_gpu_softmax_distill_rows_f32", *head, p["x"], *teacher, o["loss2"], o["top2"], o["total2"])
            go("anode_gpu_softmax_distill_bwd_rows_f32", *head, p["dy"], p["x"], *teacher, o["top2"], o["total2"], o["dx2"])
            go("anode_gpu_verify_draft_packed_f32", n, 2, 2, p["target"], p["draft"], p["token"], None, p["accept"], p["pick"],
               o["tokens"], o["accepted"])

    def scratch(self):
        q = load().symbol("anode_gpu_class_rows_scratch_bytes")
        return max(q(n, max(rows, 2), k) for n, rows, k in self.SHAPES)


def same(got, want, what):
    for a, b in zip(got, want):
        for key in a:
            assert torch.equal(a[key], b[key]), (what, key)


def test_graph_replays_equal_the_eager_result():
    chain = Chain(1)
    stream = torch.cuda.Stream()
    handle = ctypes.c_void_p(stream.cuda_stream)
    lib = load()
    stream.synchronize()
    lib.symbol("anode_gpu_release_scratch")(handle)
    assert chain.scratch() > 0 and lib.symbol("anode_gpu_reserve_scratch")(handle, chain.scratch()) == 0
    outs = chain.outputs()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        chain.run(outs, stream.cuda_stream)
    assert gpu.take_last_error() == 0
    for seed in (2, 3, 4):
        other = Chain(seed)
        for p, q in zip(chain.parts, other.parts):     # new inputs where the graph reads them
            for key in p:
                if isinstance(p[key], torch.Tensor):
                    p[key].copy_(q[key])
        want = chain.outputs()
        chain.run(want)                                # eager, on the default stream
        torch.cuda.synchronize()
        for o in outs:
            for t in o.values():
                t.fill_(-1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(outs, want, f"replay with inputs {seed}")


def test_capture_without_scratch_is_refused():
    g = np.random.default_rng(5)
    n, rows, k = 100003, 2, 9
    x, value, index = dev(logits(g, rows, n, "f32")), torch.zeros(rows * k, device="cuda"), torch.zeros(
        rows * k, dtype=torch.int32, device="cuda")
    marker = torch.zeros(4, device="cuda")
    stream = torch.cuda.Stream()
    stream.synchronize()
    load().symbol("anode_gpu_release_scratch")(ctypes.c_void_p(stream.cuda_stream))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        marker.fill_(1.0)
        rc = gpu.call("anode_gpu_top_k_rows_f32", n, rows, 0, k, 1.0, x, value, index, None)
    assert rc == 900 and gpu.take_last_error() == 900
    graph.replay()
    torch.cuda.synchronize()
    assert np.all(host(marker) == 1.0) and np.all(host(value) == 0.0)


def test_threads_on_streams_of_their_own_and_on_one():
    chains = [Chain(10 + i) for i in range(4)]
    want = []
    for c in chains:
        o = c.outputs()
        c.run(o)
        want.append(o)
    torch.cuda.synchronize()
    shared = torch.cuda.Stream()
    errors = []
    barrier = threading.Barrier(len(chains))

    def worker(i):
        try:
            stream = shared if i >= 2 else torch.cuda.Stream()
            barrier.wait()
            for rep in range(8):
                with torch.cuda.stream(stream):
                    outs = chains[i].outputs()
                    chains[i].run(outs)
                stream.synchronize()
                same(outs, want[i], f"thread {i} repetition {rep}")
        except BaseException as e:  # noqa: BLE001 - reported in the main thread
            errors.append((i, repr(e)))

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(len(chains))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_few_long_rows_in_place(kind):
    # the slots lie all over the row, the gradient overwrites the logits: loss and gradient as with separate arrays
    g = np.random.default_rng(20)
    n, rows, k = 131077, 3, 1000
    x = logits(g, rows, n, kind)
    value, index = slots(g, rows, n, k)
    dy = g.standard_normal(rows).astype(F32)
    for in_place in (True, False):
        for stride in (0, n + 51):
            check_distill(kind, x, value, index, 1.0, dy, None, "fused", stride, 0, in_place, f"in place {in_place}")
    x[1] = np.float32(torch.finfo({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kind]).min)
    check_distill(kind, x, value, index, 1.0, dy, None, "fused", 0, 0, True, "a row of lowest values")


def test_a_tensor_that_is_not_on_the_current_device_is_refused():
    with pytest.raises(ValueError, match="not on the GPU"):
        gpu.call("anode_gpu_top_k_rows_f32", 4, 1, 0, 1, 1.0, torch.zeros(4), torch.zeros(1, device="cuda"),
                 torch.zeros(1, dtype=torch.int32, device="cuda"), None)


def _pattern(rows, n, dtype):
    """Logits that depend on row and class, cheap to make on the GPU and on the host."""
    x = torch.empty(rows, n, dtype=dtype, device="cuda")
    c = torch.arange(n, device="cuda", dtype=torch.float32)
    base = ((c * 7.0) % 1021.0) * (1.0 / 128.0)
    for r in range(0, rows, 256):
        shift = torch.arange(r, min(rows, r + 256), device="cuda", dtype=torch.float32)[:, None] % 64.0
        x[r:r + 256] = base[None, :] * (1.0 + shift / 64.0)
    return x


def test_rows_beyond_2_to_the_32_elements():
    n, rows, k = 131072, 32800, 7          # 4.3e9 elements
    print("large: top_k and distill", flush=True)
    x = _pattern(rows, n, torch.bfloat16)
    assert x.numel() > 2 ** 32
    value, index = torch.empty(rows * k, device="cuda"), torch.empty(rows * k, dtype=torch.int32, device="cuda")
    norm, dy = torch.empty(rows, device="cuda"), torch.full((rows,), 1000.0, device="cuda")
    call("anode_gpu_top_k_rows_bf16", n, rows, 0, k, 1.0, x, value, index, norm)
    loss, top, total = (torch.empty(rows, device="cuda") for _ in range(3))
    picks = [0, 1, 16383, 16384, 32767, 32768, rows - 1]
    kept = x[picks].float().cpu().numpy()
    call("anode_gpu_softmax_distill_fused_fwd_bwd_rows_bf16", n, rows, 0, k, 1.0, x, value, index, norm, dy, loss, top, total, x)
    v, i = host(value).reshape(rows, k)[picks], got_u32(index).reshape(rows, k)[picks]
    want_v, want_i = ref.top_k(kept, k)
    assert np.array_equal(i, want_i) and np.array_equal(v, want_v)
    ln = host(norm)[picks]
    want_loss, want_top, want_total = ref.distill(kept, v, i, 1.0, ln)
    bound = [ref.sum_bound(r, 1.0) for r in kept]
    assert np.all(np.abs(host(loss)[picks] - want_loss) <= np.array(bound) + ref.U * np.abs(want_loss) + 1e-9)
    want_dx, q, p = ref.distill_grad(kept, v, i, 1.0, host(dy)[picks], ln)
    got = x[picks].float().cpu().numpy()
    assert np.all(np.abs(got - want_dx) <= 2.0 ** -8 * np.abs(want_dx) + 1000 * q * (1e-4) + 1000 * 4 * ref.U * p.max() + 1e-30)


def test_one_row_of_more_than_2_to_the_31_classes():
    n = 2 ** 31 + 1003
    print("large: one row", flush=True)
    x = torch.zeros(n, dtype=torch.float16, device="cuda")
    places = [5, 2 ** 31 - 1, 2 ** 31 + 5, n - 1]
    for j, c in enumerate(places):
        x[c] = 20.0 + j
    value, index, norm = torch.empty(3, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda")
    call("anode_gpu_top_k_rows_f16", n, 1, 0, 3, 1.0, x, value, index, norm)
    assert list(host(value)) == [23.0, 22.0, 21.0] and list(got_u32(index)) == [places[3], places[2], places[1]]
    s = np.exp(np.array([20.0, 21.0, 22.0, 23.0])).sum() + (n - 4)
    assert abs(host(norm)[0] - np.log(s)) <= 1e-4
    loss, top, total = (torch.empty(1, device="cuda") for _ in range(3))
    call("anode_gpu_softmax_distill_rows_f16", n, 1, 0, 3, 1.0, x, value, index, None, loss, top, total)
    p = np.exp(np.array([23.0, 22.0, 21.0]) - 23.0)
    p /= p.sum()
    want = float((p * (np.log(p) - (np.array([23.0, 22.0, 21.0]) - np.log(s)))).sum())
    assert abs(host(loss)[0] - want) <= 1e-4
    dy = torch.ones(1, device="cuda")
    call("anode_gpu_softmax_distill_bwd_rows_f16", n, 1, 0, 3, 1.0, dy, x, value, index, None, top, total, x)
    got = [float(x[c]) for c in places]
    q = np.exp(np.array([20.0, 21.0, 22.0, 23.0])) / s
    want = q - np.array([0.0, p[2], p[1], p[0]])
    assert np.all(np.abs(np.array(got) - want) <= 2.0 ** -11 * np.abs(want) + 1e-4 * q + 2.0 ** -24)
