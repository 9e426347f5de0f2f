"""CPU checks of the paged kernels' generated gfx950 code (no GPU needed): what their speed rests on and no result
shows. Decode keeps a tile's loads in flight while it works on the one before; prefill orders its LDS-DMA itself;
neither spills where the registers were counted on."""
import os
import re
import shutil
import subprocess

import pytest

import transfer_station_amd as ts
from test_paged import ATTEND
from transfer_station_amd import build as _build

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
OBJDUMP = os.path.join(ROCM, "llvm", "bin", "llvm-objdump")
READELF = os.path.join(ROCM, "llvm", "bin", "llvm-readelf")


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    """(instruction lists, spilled vector registers) by kernel name."""
    tmp = str(tmp_path_factory.mktemp("paged"))
    if not os.path.exists(_build.lib_path()):
        pytest.skip("library not built")
    if not os.access(READELF, os.X_OK) or not os.access(OBJDUMP, os.X_OK):
        pytest.skip("llvm tools not found under %s" % ROCM)
    copy = os.path.join(tmp, "lib.so")
    shutil.copy(_build.lib_path(), copy)
    subprocess.run([OBJDUMP, "--offloading", copy], cwd=tmp, check=True, stdout=subprocess.DEVNULL,
                   stderr=subprocess.DEVNULL)
    obj = os.path.join(tmp, [f for f in os.listdir(tmp) if f.endswith("gfx950")][0])
    text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", obj], check=True, stdout=subprocess.PIPE,
                          universal_newlines=True).stdout
    notes = subprocess.run([READELF, "--notes", obj], check=True, stdout=subprocess.PIPE,
                           universal_newlines=True).stdout
    funcs, cur = {}, None
    for line in text.split("\n"):
        m = re.match(r"^[0-9a-f]+ <(\S+)>:", line)
        if m:
            cur = funcs.setdefault(m.group(1), []) if "paged" in m.group(1) else None
        elif cur is not None and line.startswith("\t"):
            ins = line.strip().split("//")[0].strip()
            if ins:
                cur.append(ins)
    spills = {m.group(1): int(m.group(2)) for m in re.finditer(
        r"\.symbol: +'?(\S*?paged\S*?)\.kd'?\n(?:.*\n)*? +\.vgpr_spill_count: +(\d+)", notes)}
    return funcs, spills


def test_no_spills(code):
    spills = code[1]
    decode = {n: c for n, c in spills.items() if "paged_decode" in n}
    prefill = {n: c for n, c in spills.items() if re.search(r"paged_prefill_kernelILi(64|128)E", n)}
    assert len(decode) >= 24 and len(prefill) >= 20, (len(decode), len(prefill))
    bad = {n: c for n, c in {**decode, **prefill}.items() if c}
    assert not bad, bad


def test_decode_keeps_the_next_tiles_loads_in_flight(code):
    """Of bf16 rows, up to D = 128 and for one block of 16 rows: no wait between the products of a tile is for all
    loads. The next tile's V is asked for before this tile's scores and its K before the products with V, so four
    loads or more stay out (with two blocks of rows the compiler puts V behind half the scores, which is as fast)."""
    n = 0
    for name, ins in code[0].items():
        if not re.search(r"paged_decode_kernelILi(64|128)ELb0ELi1E", name):
            continue
        n += 1
        mf = [i for i, x in enumerate(ins) if x.startswith("v_mfma")]
        waits = [int(re.search(r"vmcnt\((\d+)\)", x).group(1)) for x in ins[mf[0] - 8:mf[-1]]
                 if x.startswith("s_waitcnt") and "vmcnt" in x]
        assert len(waits) >= 4 and min(waits) >= 4, (name, waits)
    assert n == 4, n


def test_prefill_waits_for_its_dma_at_the_end_of_a_tile(code):
    """No wait on the DMA in flight stands before an LDS read of the tile at work."""
    n = 0
    for name, ins in code[0].items():
        if not re.search(r"paged_prefill_kernelILi\d+ELb0E", name):
            continue
        n += 1
        mf = [i for i, x in enumerate(ins) if x.startswith("v_mfma")]
        bad = []
        for i in range(mf[0], mf[-1]):
            if ins[i].startswith("s_waitcnt") and "vmcnt" in ins[i]:
                nxt = [y for y in ins[i + 1:i + 6] if not y.startswith(("s_waitcnt", "s_nop"))]
                if nxt and nxt[0].startswith("ds_read"):
                    bad.append(i)
        assert not bad, (name, bad)
    assert n >= 12


def test_every_attention_kernel_is_reached(code):
    """The plans of the calls that the GPU tests make name every instance that the library holds."""
    seen = set()
    for bits, D, page, Hq, Hkv, seqs, causal, cap, slopes, mq, mk in ATTEND:
        cols = max([-(-k // page) for _, k in seqs] + [1]) + 1
        c = ts.KvCache(4096, 4096, 4096, 4096, 4096, len(seqs), cols, 1000, page, Hkv, D, bits, 4096, 4096)
        plan = ts.attn_paged_plan(c, sum(n for n, _ in seqs) + 3, Hq, causal,
                                  ts.Scores(0.0, cap, 4096 if slopes else None),
                                  mq or max([n for n, _ in seqs] + [1]), mk or max([k for _, k in seqs] + [1]))
        seen.update(k[0] for k in plan)
    held = {"attn_paged_merge_kernel<%s>" % x for n in code[0]
            for x in re.findall(r"attn_paged_merge_kernelILi(\d+)E", n)}
    for name in code[0]:
        m = re.search(r"(attn_paged_\w+?_kernel)I(Li\d+E)(Lb\dE)((?:L[ib]\d+E)+)E", name)
        if m:
            args = [m.group(2)[2:-1], "4" if m.group(3) == "Lb1E" else "16"]
            args += [x[1:] if x[0] == "i" else ("false", "true")[int(x[1:])]
                     for x in re.findall(r"L([ib]\d+)E", m.group(4))]
            held.add("%s<%s>" % (m.group(1), ", ".join(args)))
    assert len(held) >= 50 and held == seen, (sorted(held - seen), sorted(seen - held))
