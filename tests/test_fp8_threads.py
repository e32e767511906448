"""FP8 products of several threads on one stream: what a stream's launches keep is never smaller than what the launch that uses it was promised."""
import threading
import zlib

import pytest
import torch

from machx_inference_engine_b200 import ops
from machx_inference_engine_b200.ops import cuda as K
from machx_inference_engine_b200.ops.weights import from_fp8


def two_threads(monkeypatch, first, second):
    """Sizes that two calls get which want `first` and `second` bytes of an empty list, where the first call's allocation ends only after the second call has
    put its own away."""
    kept, empty, inside, done, got = [], torch.empty, threading.Event(), threading.Event(), {}

    def held(n, **kw):
        if n == first:
            inside.set()
            assert done.wait(20)
        return empty(n, **kw)

    monkeypatch.setattr(torch, "empty", held)

    def call(n):
        got[n] = K._partial_sums(kept, n, torch.device("cpu"))

    a = threading.Thread(target=call, args=(first,))
    a.start()
    assert inside.wait(20)
    call(second)
    done.set()
    a.join()
    return got[first].numel(), got[second].numel(), kept[0].numel()


@pytest.mark.parametrize("first,second", [(10, 1000), (1000, 10)])
def test_a_thread_that_allocates_late_leaves_the_larger_buffer(monkeypatch, first, second):
    a, b, left = two_threads(monkeypatch, first, second)
    assert a >= first and b >= second and left == 1000


def test_room_is_kept_and_grows():
    kept = []
    a = K._partial_sums(kept, 100, torch.device("cpu"))
    assert K._partial_sums(kept, 60, torch.device("cpu")) is a and K._partial_sums(kept, 100, torch.device("cpu")) is a
    b = K._partial_sums(kept, 101, torch.device("cpu"))
    assert b.numel() == 101 and kept[0] is b
    c = K._partial_sums(None, 50, torch.device("cpu"))
    assert c.numel() == 50 and kept[0] is b


def test_a_call_uses_the_buffer_that_it_has_checked():
    """Whatever another thread puts into the list between a call's look at it and its launch."""
    class Swapped(list):
        looks = 0

        def __getitem__(self, i):
            self.looks += 1
            return super().__getitem__(i) if self.looks == 1 else torch.empty(1, dtype=torch.uint8)

    kept = Swapped([torch.empty(100, dtype=torch.uint8)])
    assert K._partial_sums(kept, 80, torch.device("cpu")).numel() == 100


# ------------------------------------------------------------------ on the GPU
DEV = "cuda:0"


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


def product(M, N, Kd, seed):
    g = gen(M, N, Kd, seed)
    codes = (torch.randn(N, Kd, generator=g).clamp(-4, 4) * 112).to(torch.float8_e4m3fn)
    w = from_fp8(codes, (0.5 + torch.rand(-(-N // 128), -(-Kd // 128), generator=g)) * (Kd ** -0.5 / 112)).to(DEV)
    return torch.randn(M, Kd, generator=g).to(DEV, torch.bfloat16), w


@pytest.mark.gpu
def test_a_launch_refuses_too_little_room_for_its_sums(monkeypatch):
    """Before anything is launched, so nothing is written."""
    for M, kw in ((12, dict(nt=16)), (40, dict(nt=64)), (40, dict(bn=128, cuts=4))):
        x, w = product(M, 512, 2048, 0)
        out = torch.full((M, 512), 7.0, device=DEV)
        real = K._partial_sums
        monkeypatch.setattr(K, "_partial_sums", lambda kept, n, dev: real(None, n, dev)[:n - 16])
        with pytest.raises(K.KernelError):
            K._fp8_call(x, w, out, None, None, 0, 0.0, 0.0, **kw)
        monkeypatch.setattr(K, "_partial_sums", real)
        torch.cuda.synchronize()
        assert bool((out == 7).all())
        K._fp8_call(x, w, out, None, None, 0, 0.0, 0.0, **kw)
        assert not bool((out == 7).any())


@pytest.mark.gpu
def test_threads_that_start_on_a_stream_without_room():
    """Each stream is new to the library: its first calls come from threads that want different amounts of room at the same time."""
    cases = [(12, 4096, 1024), (24, 4096, 1024), (40, 1024, 4096), (100, 1024, 4096), (9, 6144, 1024)]
    work = [product(*c, i) for i, c in enumerate(cases)]
    want = [ops.linear(x, w, out_f32=True) for x, w in work]
    torch.cuda.synchronize()
    wrong = []
    for _ in range(12):
        stream = torch.cuda.Stream()
        together = threading.Barrier(len(cases))

        def run(i):
            with torch.cuda.stream(stream):
                together.wait(20)
                for _ in range(8):
                    if not torch.equal(ops.linear(*work[i], out_f32=True), want[i]):
                        wrong.append(i)

        threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        K._stream_tickets.clear()                # (streams come from a pool: the next one may be this one again)
    assert not wrong
