# SPDX-License-Identifier: Apache-2.0
"""The explicit waits of the tile kernels of k3_linear.hip, in the code that the compiler makes of them: a wait for all but the
youngest N requests leaves the stage that is read next in flight if fewer requests are younger than it than the source counts.
On the CPU, from the listing of the device code; what other waits the compiler added is not counted on."""
import os
import re
import shutil
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kimi-k3-in-c_amd")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """name -> instructions of every tile kernel."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    out = tmp_path_factory.mktemp("listing") / "k3_linear.s"
    flags = ("--offload-arch=gfx950 -O3 -std=c++17 -fPIC -w -Xclang -target-feature -Xclang -packed-fp32-ops -mllvm "
             "-amdgpu-mfma-vgpr-form --cuda-device-only -S").split()
    subprocess.run([hipcc, *flags, "-I" + os.path.join(PKG, "..", "include"), "-I" + os.path.join(PKG, "csrc"),
                    os.path.join(PKG, "csrc", "k3_linear.hip"), "-o", str(out)], check=True, capture_output=True)
    found, body = {}, None
    for line in out.read_text().split("\n"):
        line = line.split(";")[0].strip()
        m = re.match(r"(_ZN\w*lin_tile_kernel\w*):$", line)
        if m:
            body = found.setdefault(m[1], [])
        elif line.startswith(".Lfunc_end"):
            body = None
        elif body is not None and line and (not line.startswith(".") or line.startswith(".LBB")):
            body.append(line)
    return found


def is_dma(i):
    return i.startswith("buffer_load") and i.endswith(" lds")


def is_request(i):
    return i.startswith(("buffer_load", "global_load", "flat_load", "buffer_store", "global_store", "flat_store"))


def younger_dmas(code, at, n):
    """The most LDS requests there can be among the n youngest requests before instruction `at`, over all ways there."""
    label = {i[:-1]: k for k, i in enumerate(code) if i.startswith(".LBB")}
    to = {}
    for k, i in enumerate(code):
        if i.startswith(("s_cbranch", "s_branch")):
            to.setdefault(label[i.split()[1]], []).append(k)
    best, seen, todo = 0, {}, [(at, n, 0)]
    while todo:
        k, left, dmas = todo.pop()
        best = max(best, dmas)
        if left == 0 or k == 0 or seen.get((k, left), -1) >= dmas:
            continue
        seen[k, left] = dmas
        before = list(to.get(k, []))
        if not code[k - 1].startswith(("s_branch", "s_endpgm")):
            before.append(k - 1)
        for b in before:
            todo.append((b, left - is_request(code[b]), dmas + is_dma(code[b])))
    return best


def test_tile_waits(kernels):
    assert len(kernels) >= 10
    rings = 0
    for name, code in kernels.items():
        bt, bo, wt, wo, nst, wreg, _, xf32 = (int(v) for v in re.match(
            r".*lin_tile_kernelILi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELb(\d)ELi(\d+)ELb(\d)E", name).groups())
        rings += wreg
        # LDS requests of a wave in each stage: 1 KB a request
        stage = bt * (2 if xf32 else 1) // 8 // (wt * wo) + (0 if wreg else bo // 8 // (wt * wo))
        waits = 0
        for k, i in enumerate(code):
            if i != "s_barrier":
                continue
            w = next(c for c in reversed(code[:k]) if c.startswith("s_waitcnt") or is_request(c))
            m = re.search(r"vmcnt\((\d+)\)", w)
            if not m or not w.startswith("s_waitcnt"):
                continue                        # (a barrier of the epilogue)
            waits += 1
            assert younger_dmas(code, k, int(m[1])) <= (nst - 2) * stage, (name, k, w)
        assert waits >= nst, name
    assert rings == 2
