"""CPU tests of Tensor_byte and of what the 4-bit layer functions refuse."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def mt():
    import myTensor

    return myTensor


def test_bytes_are_stored_and_moved(mt):
    x = np.arange(256, dtype=np.uint8).reshape(2, 4, 32)
    t = mt.Tensor_byte(x, "cpu")
    assert t.get_shape() == [2, 4, 32] and t.Size() == 256
    assert t.numpy().dtype == np.uint8 and np.array_equal(t.numpy(), x)
    assert np.array_equal(t[1].numpy(), x[1])
    assert np.array_equal(mt.Tensor_byte(t).numpy(), x)
    assert np.array_equal(t.flatten().numpy(), x.reshape(1, -1))
    assert t.resize([3, 2]).get_data() == [0, 1, 2, 3, 4, 5]
    assert t.zeros().get_data() == [0] * 6
    assert "TinyTensor<byte>" in repr(t) and "Shape: [3, 2]" in repr(t)
    assert repr(mt.Tensor_byte(np.array([7, 65], np.uint8), "cpu")).split()[-2:] == ["7", "65"]


def test_a_byte_array_is_data_and_a_list_a_shape(mt):
    a = mt.Tensor_byte(np.array([2, 3], np.uint8), "cpu")
    assert a.get_shape() == [2] and a.get_data() == [2, 3]
    assert mt.Tensor_byte([2, 3], "cpu").get_shape() == [2, 3]
    assert mt.Tensor_byte([2, 2], "cpu", [1, 2, 255]).get_data() == [1, 2, 255, 0]


def test_bytes_have_no_arithmetic(mt):
    t = mt.Tensor_byte(np.array([1, 2, 3], np.uint8), "cpu")
    for f in (lambda: t + t, lambda: t - t, lambda: t.ones(), lambda: t.negative(), lambda: t.mults(2),
              lambda: t.floatks(1.0), lambda: t.random(0, 9), lambda: t.ReluForward(), lambda: t.ReluBackward(t),
              lambda: t.SigmoidForward(), lambda: t.SigmoidBackward(t)):
        with pytest.raises(ValueError, match="no arithmetic"):
            f()
    assert t.get_data() == [1, 2, 3]


@pytest.mark.parametrize("name", ["float", "bf16"])
def test_layers_reject_cpu_tensors(mt, name):
    import myLayer as ml

    T = getattr(mt, "Tensor_" + name)
    x, w = T([2, 64], "cpu"), T([1, 1, 1, 64], "cpu")
    c, s, n = mt.Tensor_byte([1, 1, 4, 32], "cpu"), mt.Tensor_byte([1, 1, 4, 2], "cpu"), mt.Tensor_int([1], "cpu")
    for f in (lambda: ml.QuantizeMxfp4(x, c, s), lambda: ml.DequantizeMxfp4(c, s, x, 64),
              lambda: ml.FcForwardMxfp4(x, x, c, s, x), lambda: ml.KvAppendMxfp4(w, w, c, s, c, s, n),
              lambda: ml.AttentionDecodeMxfp4(w, c, s, c, s, n, w, 0.1)):
        with pytest.raises(ValueError, match="gpu"):
            f()


def test_layers_reject_other_types(mt):
    import myLayer as ml

    c, d = mt.Tensor_byte([1, 16], "cpu"), mt.Tensor_double([1, 32], "cpu")
    with pytest.raises(TypeError):
        ml.QuantizeMxfp4(d, c, c)
    with pytest.raises(TypeError):
        ml.DequantizeMxfp4(c, d, d, 32)
