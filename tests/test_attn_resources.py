"""Occupancy of the serving engine's attention kernels as the library is built (CPU: hipcc's
resource remarks under the build's own flags)."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from smsgate_amd.ops import build


@pytest.fixture(scope="module")
def attn_resources(tmp_path_factory):
    try:
        hipcc = build.hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    out = tmp_path_factory.mktemp("kr") / "llm.o"
    r = subprocess.run([hipcc, *build.FLAGS, "-c", os.path.join(build.CSRC, "llm_kernels.hip"), "-o", str(out),
                        "-Rpass-analysis=kernel-resource-usage"], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    res, cur = {}, None
    for m in re.finditer(r"remark:\s+(.*?): (\S+) \[-Rpass", r.stderr):
        if m.group(1).strip() == "Function Name":
            cur = res.setdefault(m.group(2), {})
        else:
            cur[m.group(1).strip()] = m.group(2)
    return res


@pytest.mark.slow
@pytest.mark.parametrize("kernel,waves", [
    ("attn_prefill_st_kernelILi2ELi0E", 4),  # the default prefill attention
    ("attn_spec_kernelILi2E", 4),            # the verify step with up to 8 drafts
    ("attn_prefill_st_kernelILi1ELi0E", 5),
    ("attn_spec_kernelILi1E", 5),
    ("attn_grouped_kernelILi1ELb1E", 4),     # the decode step
])
def test_engine_attention_keeps_its_waves(attn_resources, kernel, waves):
    hits = {k: v for k, v in attn_resources.items() if kernel in k}
    assert hits, kernel
    for name, r in hits.items():
        assert int(r["Occupancy [waves/SIMD]"]) >= waves, (name, r)
        assert int(r["ScratchSize [bytes/lane]"]) == 0, (name, r)
