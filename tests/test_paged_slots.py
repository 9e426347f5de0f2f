"""The scratch of paged attention under AddressSanitizer and UndefinedBehaviorSanitizer, on the CPU: every part of
every row that calls of all kinds leave, in exactly attn_flash_scratch_bytes (tests/sanitize/paged_slots.c)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
CSRC = os.path.join(ROOT, "transfer_station_amd", "csrc")


def test_every_slot_lies_in_the_scratch(tmp_path):
    exe = str(tmp_path / "paged_slots")
    cmd = ["gcc", "-O1", "-g", "-std=gnu11", "-Wall", "-Wextra", "-fopenmp", "-fsanitize=address,undefined",
           "-fno-sanitize-recover=all", "-fno-omit-frame-pointer", "-D__HIP_PLATFORM_AMD__=1",
           "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-I" + os.path.join(ROCM, "include"),
           os.path.join(ROOT, "tests", "sanitize", "paged_slots.c"), os.path.join(CSRC, "attn_paged.c"),
           os.path.join(CSRC, "attn_flash.c"), "-lm", "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    print(r.stdout[-3000:], r.stderr[-3000:])
    assert r.returncode == 0 and "PAGED_SLOTS OK" in r.stdout
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr
