"""An infinite logit (a scaled one may overflow) has no probability to filter by: the first largest is the choice, whatever the filters."""
import subprocess
import sys

import pytest

from helpers import ROOT

CHOICE = """
import numpy as np
from kapel_b200.sampling import Sampler, Sampling
row = np.zeros(50, np.float32)
row[[7, 30]] = np.inf
print(Sampler(Sampling(temperature=0.7, seed=3, {settings})).choose(row))
"""


@pytest.mark.parametrize("settings", ["top_p=0.9", "top_k=5, top_p=0.5", "top_p=0.9, min_p=0.1", "min_p=0.1", "top_k=5", ""])
def test_the_first_infinite_logit_is_chosen(settings):
    r = subprocess.run([sys.executable, "-c", CHOICE.format(settings=settings)], capture_output=True, text=True, timeout=60, cwd=ROOT)
    assert r.returncode == 0, r.stderr
    assert int(r.stdout.split()[-1]) == 7
