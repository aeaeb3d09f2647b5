"""The shared-memory fan-in with the row finished by the host (default) and by the device (TSDF_HOST_FOLD=0)."""
import os

import numpy as np
import pytest

from tracking_sdf_amd import synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("timing", [False, True])
def test_rows_finished_by_host_or_device_give_the_same_poses_through_the_shared_segment(monkeypatch, timing):
    import tracking_sdf_amd as ts
    seq = synth.Sequence(n_frames=5, width=160, height=120, noise=True, holes=0.02, step=3)
    runs = []
    for mode in ("alone", "host", "device"):
        monkeypatch.setenv("TSDF_HOST_FOLD", "0" if mode == "device" else "1")
        s = ts.SDF(64)
        t = ts.CameraTracking(sdf=s)
        t.set_K(seq.K)
        if mode != "alone":
            s.comm_init_shm(1, 0, f"/tsdf_rows_{os.getpid()}_{mode}_{timing}")
        if timing:
            s.set_timing(True, track=True)
        poses, iters = [], []
        for k in range(5):
            xyz, nrm, rgb = seq.frame(k)
            if k > 0:
                iters.append(t.estimate_new_position(s, xyz)["iterations"])
            s.update(t, xyz, nrm, rgb)
            poses.append((t.rot.copy(), t.trans.copy()))
        buf = np.arange(30, dtype=np.float64)
        if mode != "alone":
            assert np.array_equal(s.allreduce(buf), np.arange(30, dtype=np.float64))
            s.comm_finalize()
        s.close()
        runs.append((poses, iters))
    for poses, iters in runs[1:]:
        assert iters == runs[0][1]
        for (ra, ta), (rb, tb) in zip(runs[0][0], poses):
            assert np.array_equal(ra, rb) and np.array_equal(ta, tb)
