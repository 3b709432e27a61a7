"""GPU tests of myLayer.KvGatherPaged's outputs where sequences are shorter than they are."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["float", "bf16"])
@pytest.mark.parametrize("small", [False, True])
def test_rows_without_a_key(name, small):
    """Zeros where the outputs are given their shape, in memory that held NaN; left alone where they have it."""
    import myLayer as ml
    import myTensor as mt

    rng = np.random.default_rng(3)
    T_ = getattr(mt, "Tensor_" + name)
    B, Hkv, page, d, T, L, width, npages = 4, 2, 16, 32, 40, 50, 3, 12
    k = (rng.integers(-8, 9, (B, Hkv, T, d)) / 8).astype(np.float32)  # exact in every type, under a scale of 2^-8
    pools = [(mt.Tensor_byte if small else T_)([npages, Hkv, page, d], "gpu") for _ in range(2)]
    extra = dict(k_scales=mt.Tensor_byte([npages, Hkv], "gpu"), v_scales=mt.Tensor_byte([npages, Hkv], "gpu")) if small else {}
    table = np.arange(npages, dtype=np.int32).reshape(B, width)
    table[3, 1] = -1  # a page that the pool does not have
    lengths = [40, 0, 17, 40]
    tab, n = mt.Tensor_int(table, "gpu"), mt.Tensor_int([B], "gpu", lengths)
    ml.KvAppendPaged(T_(k, "gpu"), T_(-k, "gpu"), *pools, tab, n, **extra)

    def check(out, x, rest):
        got = out.numpy().reshape(B, Hkv, L, d)
        for b, size in enumerate(lengths):
            has = np.array([j < size and table[b, j // page] >= 0 for j in range(L)])
            ref = np.full((Hkv, L, d), rest, np.float32)
            ref[:, has] = x[b][:, T - size + np.flatnonzero(has)]
            assert np.array_equal(got[b], ref)

    dirty = [T_(np.full((B, Hkv, L, d), np.nan, np.float32), "gpu") for _ in range(6)]
    del dirty  # their blocks are what the outputs get
    ko, vo = T_([1], "gpu"), T_([1], "gpu")
    ml.KvGatherPaged(*pools, tab, n, ko, vo, L, **extra)
    check(ko, k, 0.0), check(vo, -k, 0.0)
    ko, vo = (T_(np.full((B, Hkv, L, d), 3.0, np.float32), "gpu") for _ in range(2))
    ml.KvGatherPaged(*pools, tab, n, ko, vo, L, **extra)
    check(ko, k, 3.0), check(vo, -k, 3.0)
    flat = T_(np.full((B * Hkv * L * d,), np.nan, np.float32), "gpu")  # as many values, of another shape
    ml.KvGatherPaged(*pools, tab, n, flat, vo, L, **extra)
    check(flat, k, 0.0), check(vo, -k, 3.0)
    ml.KvGatherPaged(*pools, tab, n, ko, vo, 0, **extra)
    assert ko.get_shape() == [B, Hkv, 0, d]
