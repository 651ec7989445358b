"""No-GPU check of the code that the compiler makes of the product tiles' main loop: the transposing reads of LDS do not wait for the direct-to-LDS loads of later chunks."""
import re
import subprocess

from minml_amd.build import COMMON, CSRC, PRELOAD, hipcc

KERNEL = """
#include "product_tiles.hpp"
namespace mlhip
{
	void use(hipStream_t stream, const ProductPlan &plan, const Operand &a)
	{
		launch_product<half_t, Side::COLUMNS, Side::COLUMNS, false>(stream, plan, a, a, 1, PartEpilogue { nullptr, 0, 0, false });
	}
}
"""


def test_transposing_reads_wait_for_no_later_chunk(tmp_path):
    source, asm = tmp_path / "k.hip", tmp_path / "k.s"
    source.write_text(KERNEL)
    subprocess.run([hipcc()] + COMMON + PRELOAD + ["--cuda-device-only", "-S", "-I" + CSRC, str(source), "-o", str(asm)], check=True, capture_output=True)
    text = asm.read_text()
    start = re.search(r"^(_ZN5mlhip18kernel_product_256\w+):", text, re.M).end()
    code = [l.strip() for l in text[start:text.index("s_endpgm", start)].splitlines() if l.startswith("\t") and not l.strip().startswith((".", ";"))]
    multiplications = [i for i, l in enumerate(code) if l.startswith("v_mfma")]
    assert len(multiplications) == 96 and sum("ds_read_b64_tr_b16" in l for l in code) >= 96
    # the chunk that is followed by two others comes first: its 32 MFMAs hold two waits, each of which leaves a chunk's loads (8) outstanding
    loop = code[multiplications[0]:multiplications[31] + 1]
    waits = [int(n) for l in loop for n in re.findall(r"vmcnt\((\d+)\)", l)]
    assert waits and min(waits) == 8
    assert not any("scratch" in l for l in code)
