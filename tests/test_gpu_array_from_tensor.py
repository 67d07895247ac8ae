"""ConcreteNDArray over torch tensors of any layout: the values in row order, a
view where the tensor is contiguous, and the refusals of the constructor."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LAYOUTS = {"contiguous": lambda t: t, "flat": lambda t: t.view(-1), "transposed": lambda t: t.t(),
           "columns": lambda t: t[:, ::2], "a column": lambda t: t[:, 1:2], "a strided row": lambda t: t[:1, ::3],
           "flat and strided": lambda t: t.view(-1)[::5], "expanded": lambda t: t[:1].expand(4, 12),
           "permuted": lambda t: t.view(2, 3, 12).permute(2, 0, 1), "one value": lambda t: t[1, 1], "empty": lambda t: t[:0]}


@pytest.mark.parametrize("name", LAYOUTS)
def test_layouts(name):
    import torch
    import jax4j_b200 as J
    base = torch.arange(72, dtype=torch.float32, device="cuda").view(6, 12)
    t = LAYOUTS[name](base)
    a = J.ConcreteNDArray(t, tuple(t.shape))
    assert a.tensor().dim() == 1 and a.tensor().is_contiguous() and a.dtype() is J.DType.FLOAT32
    np.testing.assert_array_equal(a.numpy(), t.cpu().numpy())
    assert a.shape().size() == t.numel()
    if name in ("contiguous", "flat", "one value"):
        assert a.data_ptr() == t.data_ptr()


def test_other_types_and_refusals():
    import torch
    import jax4j_b200 as J
    b = torch.tensor([[True, False, True]])
    a = J.ConcreteNDArray(b, (1, 3))
    assert a.dtype() is J.DType.BOOL and a.tensor().is_cuda and a.numpy().tolist() == [[True, False, True]]
    a = J.ConcreteNDArray(torch.arange(4), None, J.DType.FLOAT64)
    assert a.dtype() is J.DType.FLOAT64 and a.numpy().tolist() == [0.0, 1.0, 2.0, 3.0]
    with pytest.raises(J.IllegalArgumentException, match="needs"):
        J.ConcreteNDArray(torch.zeros(4, device="cuda"), (3,))
    with pytest.raises(J.IllegalArgumentException, match="unsupported"):
        J.ConcreteNDArray(torch.zeros(4, dtype=torch.bfloat16, device="cuda"))
