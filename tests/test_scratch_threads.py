"""Calls of several host threads on one stream share its scratch without touching each other's: on the CPU against mocks
(scratch_threads.cpp), and on the GPU through the calls."""
import os
import shutil
import subprocess
import threading

import numpy as np
import pytest

from batch_ref import Batch, Dev, ints
from conftest import REPO

HIP_INCLUDE = "/opt/rocm/include"


@pytest.mark.skipif(not shutil.which("g++") or not os.path.isdir(HIP_INCLUDE), reason="needs g++ and the HIP headers")
def test_a_call_keeps_its_scratch_until_its_launches_are_made(tmp_path):
    exe = tmp_path / "scratch_threads"
    csrc = os.path.join(REPO, "tiny-llm_amd", "csrc")
    cmd = ["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", HIP_INCLUDE, "-I", csrc, os.path.join(csrc, "scratch.cpp"),
           os.path.join(REPO, "tests", "scratch_threads.cpp"), "-o", str(exe), "-lpthread"]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.endswith("all ok\n"), out.stdout + out.stderr


@pytest.mark.gpu
def test_threads_on_one_stream(gpu):
    """Adapters, split attention and projections of three requests' batches from a thread each, all on one stream and all of two launches
    over its scratch: each thread's results have the bits that they have alone."""
    stream = gpu.Stream()
    calls, outs, keep = [], [], []
    for i, (n, K, M, r) in enumerate(((3, 640, 512, 16), (40, 384, 1030, 24), (9, 1280, 96, 8))):
        b = Batch(gpu, [n, 1], [900 + n, 2500], 16, 2, 64, 1, seed=60 + i)
        T = b.tokens
        q, o = Dev(gpu, b.rng.standard_normal((T, 4, 64)), 0), Dev(gpu, np.zeros((T, 4, 64)), 0)
        attn = gpu.Attn(dtype=0, n_heads=4, q=q.ptr, out=o.ptr, scale=0.125, causal=1)
        x, y, z = (gpu.DeviceBuffer.from_array(a.astype(np.float32)) for a in (b.rng.standard_normal((T, K)), np.zeros((T, M)), np.zeros((T, M))))
        a_, b_ = Dev(gpu, b.rng.standard_normal((2, r, K)), 1), Dev(gpu, b.rng.standard_normal((2, M, r)), 1)
        sc, of = gpu.DeviceBuffer.from_array(np.float32([1, 2])), ints(gpu, [i % 2, 1])
        lora = gpu.Lora(dtype=1, n_tokens=T, in_dim=K, out_dim=M, rank=r, n_adapters=2, n_seqs=2, x=x.ptr, y=y.ptr, a=a_.ptr, b=b_.ptr, scale=sc.ptr,
                        q_start=b.d_start.ptr, adapter=of.ptr)
        w = gpu.DeviceBuffer.from_array(gpu.synth_i4(M, K, 64, seed=i))
        lib = gpu.lib()

        def call(attn=attn, b=b, lora=lora, w=w, x=x, z=z, M=M, K=K, T=T):
            return [lib.tqhip_paged_attention_dev(attn, b.c, b.s, stream.ptr), lib.tqhip_lora_add_dev(lora, stream.ptr),
                    lib.tqhip_matmul_i4_dev(w.ptr, x.ptr, z.ptr, M, K, T, 64, stream.ptr)]

        calls.append(call)
        outs.append((o.buf, T * 256, y, T * M, z, T * M))
        keep.append((q, o, x, y, z, a_, b_, sc, of, w, b, attn, lora))

    def read(o):
        return [o[i].download(np.int32, o[i + 1]) for i in (0, 2, 4)]

    want = []
    for call, o in zip(calls, outs):
        assert call() == [0, 0, 0]
        stream.synchronize()
        want.append(read(o))
    for _ in range(3):
        status = []
        go = threading.Barrier(len(calls))

        def work(call):
            go.wait()
            for _ in range(60):
                status.extend(call())

        threads = [threading.Thread(target=work, args=(c,)) for c in calls]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        stream.synchronize()
        assert not any(status) and len(status) == 3 * 60 * len(calls)
        for o, bits in zip(outs, want):
            assert all(np.array_equal(p, r) for p, r in zip(read(o), bits))
