"""`__cuda_array_interface__`: what other libraries read of an array.  No GPU: the arrays borrow an address that nothing reads."""
import pytest

import cumo_b200 as xp


def arr(*shape, T=xp.SFloat):
    return T.from_device_pointer(1 << 20, shape)


@pytest.mark.parametrize("view,shape", [(lambda: arr(4, 3), (4, 3)), (lambda: arr(1)[::-1], (1,)), (lambda: arr(4, 1)[True, ::-1], (4, 1)),
                                        (lambda: arr(6, 4)[2:3, True], (1, 4)), (lambda: arr(6, 5)[5:4:-1, True], (1, 5)), (lambda: arr(), ())])
def test_contiguous_arrays_have_no_strides(view, shape):
    """A step along an extent of 1 says nothing: the array is contiguous, also where that step is negative (which other
    libraries refuse)."""
    x = view()
    face = x.__cuda_array_interface__
    assert face["shape"] == shape and face["strides"] is None and face["data"] == (x.data_ptr, False)
    assert face["version"] == 3 and face["typestr"] == "<f4"


def test_other_arrays_have_their_steps():
    x = arr(6, 5, T=xp.DFloat)
    for v, shape, strides in ((x[::2, True], (3, 5), (80, 8)), (x.transpose(), (5, 6), (8, 40)), (x[True, 1:3], (6, 2), (40, 8))):
        face = v.__cuda_array_interface__
        assert (face["shape"], face["strides"], face["data"], face["typestr"]) == (shape, strides, (v.data_ptr, False), "<f8")
