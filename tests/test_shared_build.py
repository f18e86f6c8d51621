"""What the sources of shared prefixes and bounded caches rely on in the code that the compiler makes of them, checked on
its assembly (CPU): no vector register spills and no scratch, no packed fp32 arithmetic, and m0 (the LDS address of a
direct load, which the compiler does not know to be kept) written by nothing but the statement that uses it."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "star-kv_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")

KERNELS = {"prefix": 6 + 3 + 6 + 3 + 4,           # logits, P V, join, output, packing
           "bounded": 3 + 4 + 6 + 1}               # statistics, sums, selection, moved rows


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_no_spills_and_m0_only_where_it_is_used(name, tmp_path):
    out = tmp_path / (name + ".s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "--cuda-device-only", "-S", os.path.join(CSRC, name + ".hip"), "-o", str(out)],
                   check=True, capture_output=True)
    text = out.read_text()
    spills = re.findall(r"\.vgpr_spill_count: +(\d+)", text)
    assert len(spills) == KERNELS[name] and set(spills) == {"0"}
    assert not re.search(r"^\s+scratch_", text, re.M)
    assert not re.search(r"^\s+v_pk_(add|mul|fma)_f32", text, re.M)
    lines = [ln.split(";")[0].strip() for ln in text.splitlines()]
    lines = [ln for ln in lines if ln]
    uses = [i for i, ln in enumerate(lines) if re.search(r"\bm0\b", ln)]
    for i in uses:
        assert lines[i].startswith("s_mov_b32 m0,") and lines[i + 1] == "s_nop 0", lines[i]
        assert lines[i + 2].startswith("global_load_lds_"), lines[i:i + 3]
    assert len(uses) == sum(ln.startswith("global_load_lds_") for ln in lines)
    assert not re.search(r"^\s+(s_movrel|v_movrel|s_sendmsg|ds_append|ds_consume|ds_ordered|ds_gws|ds_read_addtid|ds_write_addtid)",
                         text, re.M)
    assert bool(uses) == (name == "prefix")
