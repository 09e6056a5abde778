# SPDX-License-Identifier: Apache-2.0
"""The layer's operators from two host threads at once, each on a stream of its own with inputs that change from pass to pass and outputs
that hold sentinels before each: what a pass leaves unwritten, or writes from another pass's or thread's data, shows."""
import threading

import pytest
import torch

from test_gpu_layer import Layer

pytestmark = pytest.mark.gpu
PASSES = 6


def say(msg):
    print(msg, flush=True)


def clear(m):
    """Sentinels in every output of the first five steps (the fill kernels of the current stream)."""
    for t in m.tensors()[:5]:
        t.fill_(-9 if t.dtype == torch.int32 else float("nan"))


@pytest.mark.parametrize("T", [3, 130, 700])
def test_fresh_outputs(gpu, k3, T):
    say(f"case: two threads, {T} tokens, {PASSES} passes each")
    ms = [Layer(k3, T, 4, 980 + i) for i in range(2)]
    sts = [torch.cuda.Stream() for _ in ms]
    wrong, want = [], []
    try:
        for i, m in enumerate(ms):
            want.append([])
            for r in range(PASSES):
                m.inputs(50 + 10 * i + r)
                clear(m)
                for s in range(5):
                    m.one(s)
                want[i].append([t.clone() for t in m.tensors()[:5]])
                assert not any(torch.isnan(t).any() for t in want[i][r] if t.dtype != torch.int32)
                assert r == 0 or not torch.equal(want[i][r][1], want[i][r - 1][1])
        xs = [[torch.randn(T, m.x.shape[1], device="cuda", generator=torch.Generator(device="cuda").manual_seed(50 + 10 * i + r))
               for r in range(PASSES)] for i, m in enumerate(ms)]
        torch.cuda.synchronize()
        start = threading.Barrier(len(ms))

        def work(i, m, st):
            try:
                got = []
                start.wait(30)
                with torch.cuda.stream(st):
                    for r in range(PASSES):
                        m.x.copy_(xs[i][r])
                        m.xr.copy_(m.x)
                        clear(m)
                        for s in range(5):
                            m.one(s, st.cuda_stream)
                        got.append([t.clone() for t in m.tensors()[:5]])
                st.synchronize()
                for r in range(PASSES):
                    for n, (g, w) in enumerate(zip(got[r], want[i][r])):
                        assert torch.equal(g, w), (i, r, n)
            except BaseException as e:
                wrong.append(e)
        th = [threading.Thread(target=work, args=(i, m, st)) for i, (m, st) in enumerate(zip(ms, sts))]
        for t in th:
            t.start()
        for t in th:
            t.join()
        assert not wrong, wrong
    finally:
        torch.cuda.synchronize()
        for m in ms:
            m.bank.free()
