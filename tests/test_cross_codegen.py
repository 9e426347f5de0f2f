"""CPU checks of cross attention's and beam search's generated gfx950 code (no GPU needed): what their speed rests on and no
result shows. The tile kernels order their LDS-DMA themselves, keep their accumulators in registers, and the library
holds no attention kernel that no call reaches."""
import os
import re
import shutil
import subprocess

import pytest

import test_cross
import transfer_station_amd as ts
from transfer_station_amd import build as _build

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
OBJDUMP = os.path.join(ROCM, "llvm", "bin", "llvm-objdump")


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    """Instruction lists by kernel, named as the plans do."""
    tmp = str(tmp_path_factory.mktemp("cross"))
    if not os.path.exists(_build.lib_path()):
        pytest.skip("library not built")
    if not os.access(OBJDUMP, os.X_OK):
        pytest.skip("llvm tools not found under %s" % ROCM)
    copy = os.path.join(tmp, "lib.so")
    shutil.copy(_build.lib_path(), copy)
    subprocess.run([OBJDUMP, "--offloading", copy], cwd=tmp, check=True, stdout=subprocess.DEVNULL,
                   stderr=subprocess.DEVNULL)
    obj = os.path.join(tmp, [f for f in os.listdir(tmp) if f.endswith("gfx950")][0])
    text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", obj], check=True, stdout=subprocess.PIPE,
                          universal_newlines=True).stdout
    funcs, cur = {}, None
    for line in text.split("\n"):
        m = re.match(r"^[0-9a-f]+ <(\S+)>:", line)
        if m:
            k = re.search(r"(attn_cross_\w*?kernel)(?:I((?:L[ib]\d+E)+)E)?", m.group(1))
            cur = None
            if k:
                args = [x[1:] if x[0] == "i" else ("false", "true")[int(x[1:])]
                        for x in re.findall(r"L([ib]\d+)E", k.group(2) or "")]
                cur = funcs.setdefault(k.group(1) + ("<%s>" % ", ".join(args) if args else ""), [])
        elif cur is not None and line.startswith("\t"):
            ins = line.strip().split("//")[0].strip()
            if ins:
                cur.append(ins)
    return funcs


def products(ins):
    mf = [i for i, x in enumerate(ins) if x.startswith("v_mfma")]
    return ins[mf[0]:mf[-1]]


def test_tiles_wait_for_their_dma_at_the_end_of_a_step(code):
    """No wait on the DMA in flight stands before an LDS read of the tile at work."""
    n = 0
    for name, ins in code.items():
        if not re.match(r"attn_cross_(dq_|dkv_)?kernel", name):
            continue
        n += 1
        hot, bad = products(ins), []
        for i, x in enumerate(hot):
            if x.startswith("s_waitcnt") and "vmcnt" in x:
                nxt = [y for y in hot[i + 1:i + 6] if not y.startswith(("s_waitcnt", "s_nop"))]
                if nxt and nxt[0].startswith("ds_read"):
                    bad.append(i)
        assert not bad, (name, bad)
    assert n == 25


def test_accumulators_stay_in_registers(code):
    """Between the products nothing goes to memory and back but, in dK and dV at D = 128, an operand of K or two."""
    for name, ins in code.items():
        if "merge" in name or "sum" in name:
            continue
        hot = products(ins)
        spilled = sum(x.startswith("scratch_") for x in hot)
        assert spilled <= (4 if "dkv_kernel<128" in name else 2), (name, spilled)


def test_every_kernel_is_reached(code):
    """The plans of the calls that the GPU tests make name every instance that the library holds."""
    seen = set()
    for seqs, Hq, Hkv, D, room, claim in test_cross.CASES:
        n, m = (max([s[i] for s in seqs] + [1]) for i in (0, 1))
        T = [max(1, room[i] * len(seqs) if room else sum(s[i] for s in seqs)) + 3 for i in (0, 1)]
        c = ts.CrossCall(ts.Spans(4096, T[0], n), ts.Spans(4096, claim or T[1], claim or m), len(seqs), Hq, Hkv, D)
        for grad in (0, 1):
            seen.update(k[0] for k in ts.attn_cross_plan(c, grad))
    assert set(code) == seen, (sorted(set(code) - seen), sorted(seen - set(code)))
