"""Build-time guards for the paged attention kernels, on their gfx950 assembly (no GPU needed).

paged_prompt_kernel addresses its tiles from LDS address 0, so it must have no LDS but what the launch asks for; over a 16-bit
cache it requests tiles straight into LDS, which the compiler does not connect with the reads behind the barrier: a wave must
have waited for its own part (vmcnt 0) before each barrier that lets the others read it. Both kernels are sized so that their
loops stay in registers."""
import os
import re
import subprocess
import tempfile

import pytest

from test_kernel_isa_cpu import CSRC, FLAGS, HIPCC, kernels, resources


def assembly(name):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    with tempfile.TemporaryDirectory() as d:
        out = os.path.join(d, name + ".s")
        subprocess.check_call([HIPCC] + FLAGS + ["-S", "--cuda-device-only", os.path.join(CSRC, name + ".hip"), "-o", out], stderr=subprocess.DEVNULL)
        return open(out).read()


@pytest.fixture(scope="module")
def prompt():
    return assembly("paged_prompt")


@pytest.fixture(scope="module")
def decode():
    return assembly("paged_decode")


def args(name):
    """activation, cache (0 fp32, 1 fp16, 2 bf16, 3 int8), head size of an instantiation"""
    return tuple(int(x) for x in re.search(r"_kernelILi(\d)ELi(\d)ELi(\d+)E", name).groups())


def test_prompt_kernel_has_no_lds_of_its_own(prompt):
    sizes = dict(re.findall(r"\.amdhsa_kernel (\S*paged_prompt_kernel\S*)\n\s*\.amdhsa_group_segment_fixed_size (\d+)", prompt))
    assert len(sizes) == 24 and set(sizes.values()) == {"0"}


def test_prompt_kernel_waits_for_its_tile_before_the_barrier(prompt):
    seen = 0
    for name, body in kernels(prompt).items():
        if "paged_prompt_kernel" not in name:
            continue
        direct = [i for i, ins in enumerate(body) if ins.startswith("global_load_lds")]
        if args(name)[1] == 3:
            assert not direct, name
            continue
        assert direct, name
        # the barriers that a tile's requests stand directly behind: the ones that open a tile
        opens = [i for i, ins in enumerate(body) if ins.startswith("s_barrier") and any(d > i for d in direct) and
                 next(x for x in body[i + 1:] if x.startswith(("global_load_lds", "s_barrier"))).startswith("global_load_lds")]
        assert len(opens) == 2, (name, len(opens))                             # two unrolled tiles
        for i in opens:
            waits = [x for x in body[max(i - 12, 0):i] if x.startswith("s_waitcnt") and "vmcnt(0)" in x]
            assert waits, (name, body[max(i - 12, 0):i + 1])
        seen += 1
    assert seen == 12


def test_loops_stay_in_registers(prompt, decode):
    """nothing in scratch memory, two workgroups (four waves each) to a CU -- three of decode's with heads of 64 --, but for fp32 queries
    (two parts each) over int8 rows of 128, which have a few registers too many"""
    for asm, kernel in ((prompt, "paged_prompt_kernel"), (decode, "paged_decode_kernel")):
        found = {n: r for n, r in resources(asm).items() if kernel in n and "NumVgprs" in r}
        assert len(found) == (48 if kernel == "paged_decode_kernel" else 24), sorted(found)
        for n, r in found.items():
            wide = kernel == "paged_prompt_kernel" and args(n) == (0, 3, 128)
            assert r["ScratchSize"] <= (64 if wide else 0), (n, r)
            assert r["NumVgprs"] + r.get("NumAgprs", 0) <= (168 if kernel == "paged_decode_kernel" and args(n)[2] == 64 else 256), (n, r)
