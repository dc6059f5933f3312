"""What the entry points of the token operators say about arguments that would otherwise reach a kernel, before anything reaches the GPU."""
import pytest

from mytorch_b200.backends.cuda.env import LIBRARY_PATH, NativeError, _binding

ADDRESS = 1 << 20  # never dereferenced


@pytest.mark.parametrize("width", [4, 6])
@pytest.mark.parametrize("count", [3, 5000])
@pytest.mark.parametrize("off", [4, 8, 12])
def test_scratch_of_the_embedding_gradient_begins_at_16_bytes(off, count, width):
    """Counts and pieces in it are read four at a time."""
    _binding.load(LIBRARY_PATH, NativeError)
    with pytest.raises(NativeError, match="16-byte"):
        _binding.embedding_backward_f32(1, ADDRESS, count, 10, width, ADDRESS, 1.0, -1, ADDRESS, ADDRESS + off, 1 << 40, None)


@pytest.mark.parametrize("hw", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 31 - 255])
def test_images_of_almost_as_many_positions_as_an_int_counts(hw):
    """The last stretch of positions ends before the largest int, or the image is refused."""
    _binding.load(LIBRARY_PATH, NativeError)
    a, big = ADDRESS, 1 << 50
    for call in (lambda: _binding.group_norm_forward_f32(1, 1, hw, 1, a, a, a, 1e-5, 0, a, a, a, a, big, None),
                 lambda: _binding.group_norm_backward_f32(1, 1, hw, 1, a, a, a, a, a, a, 0, a, a, a, a, big, None)):
        with pytest.raises(NativeError, match="too many values"):
            call()
