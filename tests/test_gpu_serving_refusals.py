"""Arguments of the serving calls that are no tensors at all raise what the documentation says (GPU)."""

import numpy as np
import pytest

from test_gpu_serving import BF16, gpu, i32, pool  # noqa: F401 (gpu: the module's fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_no_tensors(pkg):
    """NumPy arrays (what rope_tables gives), numbers, lists and tensors without dimensions for each tensor argument."""
    c, table, _ = pool(pkg, [20], 16, 2, 64, BF16, 1)
    one, zero = i32([1]), i32([0])
    kv, q = torch.zeros((1, 2, 64), device="cuda"), torch.zeros((1, 4, 64), device="cuda")
    cos, sin = (torch.from_numpy(t).cuda() for t in pkg.rope_tables(8, 64, 10000.0))
    calls = [
        (c.append, dict(k=kv, v=kv, block_table=table, seq=zero, pos=one, cos=cos, sin=sin, q=q, q_out=q.clone())),
        (c.attend, dict(q=q, block_table=table, lengths=one, seq=zero, out=q.clone(), lse=q.new_zeros((1, 4)))),
        (c.read, dict(block_table=table, seq=zero, pos=one, k_out=kv.clone(), v_out=kv.clone())),
        (pkg.token_logprobs, dict(logits=cos, tokens=torch.zeros(8, dtype=torch.int32, device="cuda"))),
    ]
    for f, good in calls:
        f(**good)
        for name in good:
            for odd in (3, "x", [1.0], np.zeros((1, 2, 64), np.float32), np.zeros(1, np.int32), torch.zeros(()),
                        torch.zeros((), device="cuda"), torch.zeros((), dtype=torch.int32, device="cuda")):
                with pytest.raises(ValueError):
                    f(**{**good, name: odd})
                    pytest.fail(f"{f.__name__} took {odd!r} for {name}")
    with pytest.raises(ValueError):
        c.append(kv, kv, table, zero, one, *pkg.rope_tables(8, 64, 10000.0), q=q)
    for odd in ("x", [1.0]):
        with pytest.raises((ValueError, TypeError)):
            c.attend(q, table, one, sm_scale=odd)
