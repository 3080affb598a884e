"""MXFP4 and few-token calls of several threads at once: the bits of one call alone, every call made and
none ended by an error."""
import threading
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch


def together(work, n):
    """work(0) .. work(n - 1) in threads that start at once; their results, or the first one's error."""
    start = threading.Barrier(n, timeout=60)

    def run(k):
        start.wait()
        return work(k)

    with ThreadPoolExecutor(n) as pool:
        return [f.result() for f in [pool.submit(run, k) for k in range(n)]]


def test_an_error_in_a_thread_is_raised():
    assert together(lambda k: k * k, 4) == [0, 1, 4, 9]
    with pytest.raises(ZeroDivisionError):
        together(lambda k: 1 // (k - 2), 4)


@pytest.mark.gpu
@pytest.mark.parametrize("own", [False, True])
def test_calls_of_threads(gpu_device, own):
    """On one stream and on their own; rows of one launch, of the quantizer's and of a tiled product."""
    from kb_nano_amd import FewTokenExperts, Mxfp4Linear, Mxfp4Quant, dequantize_mxfp4
    print(f"mxfp4 threads own={own}", flush=True)
    quant, lin, few = Mxfp4Quant(), Mxfp4Linear(), FewTokenExperts()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(300, 512, generator=g).bfloat16().to(gpu_device)
    w, sw = quant((torch.randn(4, 512, 512, generator=g) * 0.05).to(gpu_device))
    w2, s2 = w[:, :, :128].contiguous(), sw[:, :, :8].contiguous()
    ids = torch.randint(0, 4, (40, 2), generator=g).to(torch.int32).to(gpu_device)
    tw = torch.rand(40, 2, generator=g).to(gpu_device)

    def calls(n):
        m = min(n, 40)
        c, s = quant(x[:n])
        return (lin(x[:n], w[0], sw[0]), lin(x[:n].float(), w[1], sw[1]), few(x[:m], w, w2, tw[:m], ids[:m], 4, sw, s2, [1, 32]),
                c, s, dequantize_mxfp4(c, s))

    rows = (1, 7, 40, 300)
    refs = [calls(n) for n in rows]
    torch.cuda.synchronize()

    def work(k):
        made = 0
        stream = torch.cuda.Stream() if own else torch.cuda.current_stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                outs = calls(rows[k])
                assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(outs, refs[k], strict=True))
                made += len(outs)
        return made

    assert together(work, len(rows)) == [30 * 6] * len(rows)
    torch.cuda.synchronize()
