"""What the library's kernels ask of the hardware, compiled with the library's own flags: no scratch memory (a kernel that has a
private segment starts about a microsecond later) and no packed fp32 instruction (some of their forms have given wrong results here)."""
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

from distributed_tensorflow_amd import build

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")
@pytest.mark.timeout(900)
def test_the_shipped_kernels_use_no_scratch_and_no_packed_fp32(tmp_path):
    def assembly(src):
        out = tmp_path / (src.stem + ".s")
        flags = [f for f in build.HIP_FLAGS if f not in ("-fPIC", "-Wall")]
        subprocess.run([HIPCC, *flags, f"-I{build.CSRC}", "--cuda-device-only", "-S", str(src), "-o", str(out)], check=True,
                       stderr=subprocess.DEVNULL)
        return out.read_text()

    sources = sorted(build.CSRC.glob("*.hip"))
    with ThreadPoolExecutor(max_workers=8) as pool:
        texts = dict(zip(sources, pool.map(assembly, sources)))
    kernels = [(src.name, name, int(size)) for src, text in texts.items() for name, size in
               re.findall(r"\.amdhsa_kernel (\S+).*?\.amdhsa_private_segment_fixed_size (\d+)", text, flags=re.S)]
    assert len(kernels) >= 10
    assert not [k for k in kernels if k[2]]
    assert not [(src.name, op) for src, text in texts.items() for op in re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", text)]
