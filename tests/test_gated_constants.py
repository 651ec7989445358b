"""No-GPU check of the coefficients in the gated layer's kernels: the tail of the normal distribution as fp16 takes it."""
import os
import re

import numpy as np
from scipy.special import erfcx

from minml_amd.build import CSRC


def test_tail_of_the_normal_distribution():
    """t P(t) exp(-z^2) with t = 1 / (1 + 0.43 z) against 0.5 erfc(z): 2.53e-6 relative, everywhere in z = 0 .. 7, as the comment beside it says."""
    text = open(os.path.join(CSRC, "gated.hip")).read()
    body = text[text.index("float normal_tail(float g)"):text.index("0.5f * erfcf")]
    scale = float(re.search(r"fabsf\(g\), ([0-9.]+)f \* 0.70710678", body).group(1))
    first = re.search(r"fmaf\(t, (-?[0-9.]+)f, (-?[0-9.]+)f\)", body)
    coefficients = [float(first.group(1)), float(first.group(2))] + [float(c) for c in re.findall(r"fmaf\(t, poly, (-?[0-9.]+)f\)", body)]
    assert len(coefficients) == 6
    z = np.linspace(0, 7, 20001)
    t = 1 / (1 + scale * z)
    relative = t * np.polyval(coefficients, t) / (0.5 * erfcx(z)) - 1
    assert np.abs(relative).max() <= 2.54e-6
