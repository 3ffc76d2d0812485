"""Sizes whose launch would be 2^32 threads and more are refused: such a launch runs the rest beyond 2^32 only and reports no error.  No GPU, no
launch: the refusal comes first."""
import pytest

from lbm_amd import _lib

P = 4096      # stands for a device pointer in calls that are refused before it is used
R = 1 << 26   # rows of four to a workgroup of 256 threads
CALLS = {
    "lbm_bandpower_f32": lambda lib, n: lib.lbm_bandpower_f32(P, P, P, n, 1, 27, 1, 0, None),
    "lbm_rownorm2_f32": lambda lib, n: lib.lbm_rownorm2_f32(P, P, n, 4, None),
    "lbm_epochs_gather_f32": lambda lib, n: lib.lbm_epochs_gather_f32(P, 1000, P, P, n, 1, 10, 1000, None),
    "lbm_channel_scale_f32": lambda lib, n: lib.lbm_channel_scale_f32(P, P, P, P, n, 1, 8, None),
    "lbm_channel_moments_f32": lambda lib, n: lib.lbm_channel_moments_f32(P, None, P, P, n, 1, 8, None),
    "lbm_epoch_post_f32": lambda lib, n: lib.lbm_epoch_post_f32(P, P, P, None, n, 1, 1500, 0, 1.0, 0, 0.0, None),
    "lbm_affine_ch_f32": lambda lib, n: lib.lbm_affine_ch_f32(P, P, n, 4, 4, 8, P, P, None),
    "lbm_affine_post_f32": lambda lib, n: lib.lbm_affine_post_f32(P, P, P, P, P, None, None, n, 4, 4, 64, 0, 1.0, 0, 0.0, None),
    "lbm_fir_f32": lambda lib, n: lib.lbm_fir_f32(P, P, n, 64, P, 5, 0, None),
    "lbm_welch_f32": lambda lib, n: lib.lbm_welch_f32(P, P, None, n, 255, 250.0, 255, 200, 100, P, 0, 20, 0, None),
    "lbm_vq_argmin_f32": lambda lib, n: lib.lbm_vq_argmin_f32(P, 8, 0, 0, P, P, P, None, None, n, 8, 16, None),
    "lbm_conv1d_f32": lambda lib, n: lib.lbm_conv1d_f32(P, P, P, P, n, 3, 64, 5, 5, 1, 2, 0, None),
}
# the first size that is refused
FIRST = {"lbm_bandpower_f32": R - 3, "lbm_rownorm2_f32": R - 3, "lbm_epochs_gather_f32": R - 3, "lbm_channel_scale_f32": R - 3,
         "lbm_channel_moments_f32": R - 3, "lbm_epoch_post_f32": R - 3, "lbm_affine_ch_f32": 1 << 25, "lbm_affine_post_f32": 1 << 26,
         "lbm_welch_f32": 1 << 24, "lbm_fir_f32": (1 << 32) // 192 + 1, "lbm_vq_argmin_f32": ((1 << 24) - 1) * 128 + 1}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_launches_of_two_to_the_32_threads_are_refused(name):
    lib = _lib.load()
    for n in (FIRST.get(name, 1 << 36), 1 << 36, 1 << 40):
        assert CALLS[name](lib, n) == -2, n
        assert name.replace("_f32", "") in lib.lbm_last_error().decode()
