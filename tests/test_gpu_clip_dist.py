"""GPU (-m gpu): a clipped iteration of a view-sharded job.  Every rank clips by the norm of the exchanged gradients: the ranks
hold the same state after every iteration, and two ranks with one view each end where one process averaging the two views
ends, bit for bit -- with the SH gradient as factors (which enter the norm without being written) and dense, through an
iteration that densifies (whose new tensors have no gradients) and one that resets the opacities.  The ranks share the one GPU
and talk over gloo, as in test_gpu_dist_train.py."""
import hashlib
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))
BOUND, STEPS = 2e-4, 4

WORKER = r"""
import sys
sys.path.insert(0, %(root)r); sys.path.insert(0, %(root)r + "/tests")
import numpy as np, torch
from vegs_amd import dist as vdist
import test_gpu_clip_dist as me
rank, world, local = vdist.init_from_env()
torch.cuda.set_device(0)
digests, norms, state = me.train(world, rank, %(exchange)r)
np.savez(%(out)r + "/rank%%d.npz" %% rank, digests=np.array(digests), norms=np.array(norms), **state)
torch.distributed.barrier()
torch.distributed.destroy_process_group()
print("RANK_OK", rank)
"""


def train(world, rank, exchange):
    import dist_train_case as case
    tr, deg, cams, gts, normals = case.make(world, rank, exchange, torch.device("cuda", 0), P=20000)
    tr.max_grad_norm = BOUND
    digests, norms = [], []

    def on_step(it, tr):
        h = hashlib.sha256()
        for k, v in sorted(case.state_numpy(tr).items()):
            h.update(k.encode())
            h.update(np.ascontiguousarray(v).tobytes())
        digests.append(h.hexdigest())
        norms.append(float(tr.last["grad_norm"]))

    case.run(tr, deg, cams, gts, normals, STEPS, 2, world, rank, on_step)
    return digests, norms, case.state_numpy(tr)


@pytest.mark.parametrize("exchange", ["factored", "dense"])
def test_two_ranks_clip_as_one_process_does(tmp_path, exchange):
    from test_gpu_dist_train import _free_port
    from vegs_amd import rasterizer
    script, port, procs = WORKER % dict(root=ROOT, exchange=exchange, out=str(tmp_path)), _free_port(), []
    for r in range(2):
        env = dict(os.environ, RANK=str(r), WORLD_SIZE="2", LOCAL_RANK=str(r), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port),
                   VEGS_DIST_BACKEND="gloo")
        procs.append(subprocess.Popen([sys.executable, "-c", script], env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                      text=True))
    outs = [p.communicate(timeout=100)[0] for p in procs]
    assert all(p.returncode == 0 for p in procs) and all("RANK_OK" in o for o in outs), "\n".join(o[-3000:] for o in outs)
    ranks = [np.load(tmp_path / f"rank{r}.npz") for r in range(2)]
    old = rasterizer.get_flags()
    try:
        _, norms, want = train(1, 0, exchange)
    finally:
        rasterizer.set_flags(old)
    assert list(ranks[0]["digests"]) == list(ranks[1]["digests"]) and len(ranks[0]["digests"]) == STEPS
    assert np.isfinite(norms).all() and norms[0] > BOUND                     # it did clip
    assert list(ranks[0]["norms"]) == norms and list(ranks[1]["norms"]) == norms
    bad = [k for k in sorted(want) if not np.array_equal(ranks[0][k], want[k])]
    assert not bad, bad[:8]
