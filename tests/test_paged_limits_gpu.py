"""The paged cache's entry points at the limits of what they take."""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def mt():
    import mytorch_b200 as m
    return m


def child(code):
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    return run.stdout


# The kernel's shared memory is 8 bytes a request and 512 besides: 48 KB, where a launch has to ask for more, lies at 6080
# requests. Each first in a process of its own, as one call that asked helps all later ones.
@pytest.mark.parametrize("requests", [6080, 6081, 6144, 6145, 8192])
def test_tables_as_a_process_first_call(requests):
    child("import numpy as np, mytorch_b200 as mt, tests.test_paged_gpu as t;"
          f"t.check_tables(mt, np.full({requests}, 15), np.full({requests}, 2), 16, 2, {requests}, {2 * requests})")
