"""CPU check of the arrivals of the paged attention kernels and of the per-row
sampling kernel in their compiled gfx950 assembly: what a block leaves for the
last one has completed, for every wave of it, before its arrival is counted.  The
attention kernels store partials at agent scope; k_sr_pick lists candidates and
masses with agent-scope stores."""
import os
import re
import shutil
import subprocess

import pytest

from test_isa_arrival import ARRIVE, BARRIER, ROOT, WAIT0, arrival_problems, kernel_asm

WRITE = re.compile(r"^\s*global_(store|atomic)_\w+")


def order_problems(asm: str):
    """Faults of the last arrival of a kernel: the write before it (a store at agent
    scope or an atomic) is waited for, then the block meets, then it arrives."""
    lines = [l for l in asm.split("\n") if l.strip() and not l.strip().startswith(";")]
    arrivals = [i for i, l in enumerate(lines) if ARRIVE.match(l)]
    if not arrivals:
        return ["no arrival"]
    a = arrivals[-1]
    writes = [i for i in range(a) if WRITE.match(lines[i])]
    if not writes:
        return ["no write before the arrival"]
    out = []
    if "store" in lines[writes[-1]] and "sc1" not in lines[writes[-1]]:
        out.append("store without sc1: " + lines[writes[-1]].strip())
    between = lines[writes[-1] + 1:a]
    wait = next((k for k, l in enumerate(between) if WAIT0.match(l)), None)
    if wait is None:
        out.append("no s_waitcnt vmcnt(0) after the last write")
    elif not any(BARRIER.match(l) for l in between[wait:]):
        out.append("no s_barrier after the wait")
    if not any("sc1" in l and "global_load" in l for l in lines[a:]):
        out.append("nothing read at agent scope after the arrival")
    return out


def test_detector_catches_misorderings():
    good = ("\tglobal_atomic_add_x2 v0, v[2:3], s[0:1]\n\ts_waitcnt vmcnt(0)\n\ts_barrier\n"
            "\tglobal_atomic_add v3, v3, v4, s[2:3] sc0\n"
            "\tglobal_load_dword v5, v6, s[0:1] sc1\n")
    assert order_problems(good) == []
    for bad in (good.replace("\ts_waitcnt vmcnt(0)\n", ""), good.replace("\ts_barrier\n", ""),
                good.replace(" sc1", ""),
                good.replace("global_atomic_add_x2 v0, v[2:3]", "global_store_dword v0, v2")):
        assert order_problems(bad), bad


@pytest.fixture(scope="module")
def asm_of(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    from neonengine_amd import _build
    flags = [f for f in _build.HIPCC_FLAGS if f != "-shared"]
    texts = {}

    def get(name):
        if name not in texts:
            src = os.path.join(ROOT, "neonengine_amd", "csrc", name + ".hip")
            out = tmp_path_factory.mktemp("isa") / (name + ".s")
            subprocess.run([hipcc] + flags + ["-I", os.path.join(ROOT, "include"),
                                              "--cuda-device-only", "-S", src, "-o", str(out)],
                           check=True, capture_output=True, timeout=900)
            texts[name] = out.read_text()
        return texts[name]

    return get


@pytest.mark.parametrize("kernel", ["k_paged_attn_few", "k_paged_attn_many"])
@pytest.mark.parametrize("form", ["ILi64ELb0E", "ILi64ELb1E", "ILi128ELb0E", "ILi128ELb1E"])
def test_paged_attention_arrival_order(asm_of, kernel, form):
    problems = arrival_problems(kernel_asm(asm_of("neon_paged"), kernel + form))
    assert problems == [], problems[:4]


def test_sample_rows_arrival_order(asm_of):
    problems = order_problems(kernel_asm(asm_of("neon_sample_rows"), "k_sr_pick"))
    assert problems == [], problems
