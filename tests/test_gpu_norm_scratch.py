"""The norms' gradient writes to the scratch that it asks for and not behind it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
BEHIND = 1 << 14


@pytest.mark.parametrize("gate", [None, "channel", "sample", "full"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 5), (2, 33), (7, 96), (3, 40, 64), (64, 9, 130), (5, 1, 1023), (2, 3, 1024), (40, 50, 512), (9, 8192), (3, 70, 2049), (2, 9, 10004), (1, 16386),
                                   (3, 5, 33000), (700, 3, 40), (2000, 2, 8)])
def test_nothing_behind_the_scratch(monkeypatch, shape, gate):
    import gpu_util as g
    from mytorch_b200.backends.cuda.env import CudaEnv, CudaMemory

    rng = np.random.default_rng(1)
    c = shape[-1]
    gates = {None: None, "channel": (c,), "sample": (shape[0], c), "full": shape}[gate]
    x, b, dnew, dy = (g.dev(rng.standard_normal(shape).astype(np.float32)) for _ in range(4))
    w, pw = (g.dev(rng.standard_normal(c).astype(np.float32)) for _ in range(2))
    gt = None if gates is None else g.dev(rng.standard_normal(gates).astype(np.float32))
    new, y, rstd, block_rstd = g.op("add_rms_norm")(x, b, w, pw, gt)
    call = lambda: [g.host(t) for t in g.op("add_rms_norm_backward")(dnew, dy, new, rstd, block_rstd, x, b, w, pw, gt) if t is not None]
    want = call()

    env, given = CudaEnv.instance(), []

    def workspace(nbytes):
        memory = CudaMemory(0, nbytes + BEHIND)
        memory.write(np.full(nbytes + BEHIND, 0x5A, np.uint8))
        given.append((memory, nbytes))
        return memory.ptr, nbytes

    monkeypatch.setattr(env, "workspace", workspace)
    got = call()
    (memory, nbytes), = given
    assert (memory.read((nbytes + BEHIND,), np.uint8)[nbytes:] == 0x5A).all()
    assert len(got) == len(want) and all(np.array_equal(p, q) for p, q in zip(got, want))
