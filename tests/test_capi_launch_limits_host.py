"""What a launch cannot take is refused before any of a call's kernels runs. No kernel is launched here."""
from test_capi_recurrent_host import FAKE, _lr, lib  # noqa: F401


def test_calls_past_a_launch_of_the_recurrence_are_refused(lib):  # noqa: F811
    # the workgroups are numbered in 32 bits
    most = dict(n_seq=(1 << 31) - 1, n_tokens=(1 << 31) - 1, seq_len=1, workspace=FAKE, workspace_bytes=1 << 60)
    assert lib.lampa_lr_slots(_lr(**most, D=1, x_stride=1, decay_stride=1)) == (1 << 31) - 1
    back = dict(dy=FAKE, dx=FAKE, ddecay=FAKE, dA=FAKE, tile_states=FAKE)
    odd = dict(most, D=65, x_stride=65, decay_stride=65)  # two workgroups over the channels
    assert lib.lampa_lr_scan_fwd(_lr(**odd), None) == -4 and lib.lampa_lr_scan_bwd(_lr(**odd, **back), None) == -4
