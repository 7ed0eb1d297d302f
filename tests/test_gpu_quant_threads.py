"""The 8-bit operators from several threads at once, each on its own stream:
every result equals the one made alone."""

import threading

import pytest

from test_gpu_quant_linear import operands, rng
from test_gpu_residual_norm import make

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_threads_on_their_own_streams():
    from rns8_b200 import quant

    def job(seed):
        m = (3, 70, 700, 1500)[seed]
        _, _, w, ws, b = operands(1, 2 * 520, 1040, seed)
        x = torch.randn(m, 1040, generator=rng(seed), device="cuda").to(torch.bfloat16)
        t = make(m, 1040, 1, torch.bfloat16, seed=seed)
        args = {k: t[k] for k in ("post_weight", "pre_weight", "gate")}

        def run():
            rows = quant.linear(x, w, ws / 32, bias=b, gated=True, quantize=True)
            y = quant.linear(rows, w[:, :520], ws)  # weights off 16 bytes: copied in scratch
            xo, h = quant.residual_norm(**t)
            return (*rows[:2], y, xo, h, *quant.residual_norm_backward(h, xo, xo, t["y"], **args))

        return run

    jobs = [job(s) for s in range(4)]
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    start, failures = threading.Barrier(4), []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(20):
                    got = jobs[i]()
                    stream.synchronize()
                    failures.extend((i, k) for k, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
        except Exception as e:  # noqa: BLE001
            failures.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[:5]
    quant.check_status(0)
