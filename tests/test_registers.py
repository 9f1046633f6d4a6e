"""The kernels that keep accumulators in registers written by inline-asm MFMAs must not
spill: the compiler does not know those instructions' latency, and a spill's copy of an
accumulator right behind one reads it before it is written."""
import re
import subprocess

import pytest

import __graft_entry__ as ge


@pytest.mark.parametrize("source", ["attn_prefill", "attn_paged_prefill"])
def test_kernels_with_asm_accumulators_do_not_spill(source, tmp_path):
    builder = ge._load_builder()
    csrc = next(p for p in ge.PKG_DIR.rglob(f"{source}.hip"))
    out = tmp_path / "out.s"
    subprocess.run([builder.hipcc(), *builder.HIPCC_FLAGS, *builder.FILE_FLAGS.get(source, []),
                    "--cuda-device-only", "-S", str(csrc), "-o", str(out)],
                   check=True, capture_output=True, timeout=300)
    text = out.read_text()
    found = 0
    for entry in re.split(r"^  - (?=\.)", text[text.index("amdhsa.kernels"):], flags=re.M)[1:]:
        name = re.search(r"\.name: +(\S+)", entry).group(1)
        body = text[text.index(f"\n{name}:"):]
        if "v_mfma" in body[:body.index(".Lfunc_end")].split("#APP", 1)[-1]:
            assert re.search(r"\.vgpr_spill_count: +0\b", entry), f"{name} spills"
            found += 1
    assert found >= 3
