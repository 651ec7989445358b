"""No-GPU check of the code that the compiler makes of layer normalisation: rows that are said to lie in registers do."""
import os
import re
import subprocess

from minml_amd.build import COMMON, CSRC, PRELOAD, hipcc


def test_no_kernel_of_layer_normalisation_spills(tmp_path):
    run = subprocess.run([hipcc()] + COMMON + PRELOAD + ["-Rpass-analysis=kernel-resource-usage", "--cuda-device-only", "-c", os.path.join(CSRC, "layernorm.hip"), "-o", str(tmp_path / "k.o")],
                         check=True, capture_output=True, text=True)
    names = re.findall(r"Function Name: (\S+)", run.stderr)
    scratch = re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", run.stderr)
    assert len(names) == len(scratch) and sum("kernel_layer_norm_backward" in n for n in names) >= 20
    assert {n: s for n, s in zip(names, scratch) if s != "0"} == {}
