"""The layer operators called from several threads."""

import threading

import pytest
import torch

import pearl_b200 as pg
from tests.test_gpu_layer_ops import BF16, gen, int8

pytestmark = pytest.mark.gpu


def test_products_from_several_threads():
    """Each thread on its own stream, products of pair tiles of both widths and
    of single CTAs: what is looked up once a device is not torn."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    g = gen(1)
    cases = []
    for m, n, k in ((1024, 1024, 512), (300, 2048, 256), (40, 512, 256)):
        A, B = int8(g, m, k), int8(g, n, k)
        sa, sb = torch.ones(m, device="cuda"), torch.full((n,), 1e-4, device="cuda")
        want = torch.empty(m, n, dtype=BF16, device="cuda")
        pg.gemm_epilogue(A, B, sa, sb, want)
        cases.append((A, B, sa, sb, want))
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(4)

    def work(at):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            for i in range(30):
                A, B, sa, sb, want = cases[(at + i) % 3]
                C = torch.empty_like(want)
                pg.gemm_epilogue(A, B, sa, sb, C)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(C, want):
                    wrong.append((at, i))

    threads = [threading.Thread(target=work, args=(at,)) for at in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
