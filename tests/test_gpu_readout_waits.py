"""What becomes of a readout kernel's wait that runs out: every caller learns of it, and no other launch suffers."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def lost(T):
    """A context that has lost a wait (a kernel's, on a barrier that nothing arrives on, about two seconds)."""
    ctx = T.default_context(0)
    T.quantize_rows(torch.ones(1, 16, device="cuda"))
    torch.cuda.synchronize()

    def lose():
        T._ffi.check(T.lib().thrml_debug_lose_wait(ctx.h, torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
    yield lose
    torch.cuda.synchronize()
    ctx.reset_waits()


def calls(T):
    x = torch.ones(2, 32, device="cuda")
    w, one = torch.ones(3, 32, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")
    i = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    return [lambda: T.quantize_rows(x), lambda: T.int8_linear(x, w, one), lambda: T.int8_matmul(w, one, w, one), lambda: T.adjust_logits(x), lambda: T.draw_categories(x, 1),
            lambda: T.distill_loss(x, i, x[:, :1]), lambda: T.distill_step(x, i, x[:, :1]), lambda: T.default_context(0).synchronize()]


def test_every_caller_learns_of_a_lost_wait(T, lost):
    every = calls(T)
    lost()
    failures = []

    def ask():
        for f in every:
            with pytest.raises(T.ThrmlError, match="gave up waiting") as e:
                f()
            failures.append(e.value.code)
    other = threading.Thread(target=ask)
    ask()  # a first answer does not take the report from the next, nor from another thread
    other.start()
    other.join()
    assert failures == [-5] * (2 * len(every))
    T.default_context(0).reset_waits()
    for f in every:
        f()
    torch.cuda.synchronize()


@pytest.mark.parametrize("m, k, n", [(1, 4096, 513), (16, 4096, 300), (33, 784, 4097), (700, 2000, 5000), (1280, 131071, 2048)])  # split K, one tile a CTA, pairs, waits of hundreds of microseconds
def test_a_lost_wait_ends_no_other_launch(T, lost, m, k, n):
    """A captured product that is replayed after the loss gives what it gave before."""
    g = torch.Generator("cuda").manual_seed(m)
    rows = lambda r: torch.randint(-127, 128, (r, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]  # noqa: E731
    a, w = rows(m), rows(n)
    qs, ws = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
    out = torch.zeros(m, n, device="cuda")
    want = T.int8_matmul(a, qs, w, ws)
    x = torch.randn(m, k, generator=g, device="cuda") if m <= 64 else None
    want_x = None if x is None else T.int8_linear(x, w, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        T.int8_matmul(a, qs, w, ws, out=out)
        out_x = None if x is None else T.int8_linear(x, w, ws)
    lost()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (x is None or torch.equal(out_x, want_x))


def test_two_threads_of_a_context(T):
    """Products on two threads and streams at once, with first calls of kernels among them, are each their own."""
    sets = []
    for seed in range(2):
        g = torch.Generator("cuda").manual_seed(seed)
        sets.append([(torch.randn(m, k, generator=g, device="cuda"), *T.quantize_rows(torch.randn(n, k, generator=g, device="cuda"))) for m, k, n in ((1, 512, 300), (20, 1000, 77), (50, 640, 4000), (400, 300, 9000))])
    want = [[T.int8_linear(*a) for a in s] for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                for a, b in zip(sets[i], want[i]):
                    if not torch.equal(T.int8_linear(*a), b):
                        wrong.append(i)
        stream.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("m, k, n", [(3, 100, 300), (20, 1000, 777), (64, 512, 5000), (700, 640, 9000)])  # one or two launches, K split, pairs
def test_one_workspace_for_call_behind_call(T, m, k, n):
    """The product takes the scales that the quantiser of its own call wrote, though both are at work at once and all calls share their workspace."""
    g = torch.Generator("cuda").manual_seed(m)
    w, ws = T.quantize_rows(torch.randn(n, k, generator=g, device="cuda"))
    xs = [torch.randn(m, k, generator=g, device="cuda") * 10.0**i for i in range(-6, 6)]
    want = [T.int8_matmul(*T.quantize_rows(x), w, ws) for x in xs]
    pitch = (k + 15) // 16 * 16
    q, scale = torch.empty(m, pitch, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    outs = [torch.empty(m, n, device="cuda") for _ in xs]
    h, stream = T.default_context(0).h, torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    for _ in range(5):
        for x, out in zip(xs, outs):
            T._ffi.check(T.lib().thrml_linear_i8(h, stream, m, n, k, x.data_ptr(), 0, k, q.data_ptr(), pitch, scale.data_ptr(), w.data_ptr(), w.stride(0), ws.data_ptr(), None, out.data_ptr(), 0, n))
        torch.cuda.synchronize()
        for out, v in zip(outs, want):
            assert torch.equal(out, v)
            out.zero_()
