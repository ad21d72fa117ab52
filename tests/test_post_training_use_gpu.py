"""Post-training steps on a GPU run through the kernels of their losses."""
import os
import subprocess
import sys

import pytest

from common import ROOT, free_port

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["dpo", "clipped", "reference", "moe"])
def test_post_training_steps_run_their_kernels(kind):
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT=str(free_port()), WORLD_SIZE="1", RANK="0", LOCAL_RANK="0")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "workers", "post_training_kernels_worker.py"), kind], env=env,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "KERNELS_OK" in r.stdout, (r.stdout + r.stderr)[-4000:]
