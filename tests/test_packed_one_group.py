"""A group size of 0 stands for one group of all columns, as in the quantizer's configuration."""
import ctypes

import pytest

import conftest  # noqa: F401  (import paths)


def test_bytes_of_one_group():
    import cdclq

    lib = cdclq.lib()
    gb = (ctypes.c_uint8 * 1)(3)
    assert lib.cdclq_packed_layer_bytes(16, 200, 0, gb) == lib.cdclq_packed_layer_bytes(16, 200, 200, gb) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("t", [3, 40])
def test_one_group(gpu, t):
    from cdclq import CdclqError
    from cdclq import adapters as A
    from test_gpu_adapters import layer, tokens

    (q, s, z, perm, gb, g), _ = layer(40, 200, [3], 0, 7)
    x, _ = tokens(t, 200, 1, "bf16", 1)
    assert bool((A.forward(x, A.PackedProjection(q, s, z, perm, gb, 0)) == A.forward(x, A.PackedProjection(q, s, z, perm, gb, g))).all())
    with pytest.raises(CdclqError, match="one width"):
        A.PackedProjection(q, s, z, perm, gb, -1)
