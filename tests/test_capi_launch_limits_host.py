"""What a launch cannot take is refused before any of a call's kernels runs. No kernel is launched here."""
from test_capi_recurrent_host import FAKE, _ff, _lr, lib  # noqa: F401


def test_calls_past_a_launch_of_the_recurrence_are_refused(lib):  # noqa: F811
    # the workgroups are numbered in 32 bits
    most = dict(n_seq=(1 << 31) - 1, n_tokens=(1 << 31) - 1, seq_len=1, workspace=FAKE, workspace_bytes=1 << 60)
    assert lib.lampa_lr_slots(_lr(**most, D=1, x_stride=1, decay_stride=1)) == (1 << 31) - 1
    back = dict(dy=FAKE, dx=FAKE, ddecay=FAKE, dA=FAKE, tile_states=FAKE)
    odd = dict(most, D=65, x_stride=65, decay_stride=65)  # two workgroups over the channels
    assert lib.lampa_lr_scan_fwd(_lr(**odd), None) == -4 and lib.lampa_lr_scan_bwd(_lr(**odd, **back), None) == -4


def test_calls_past_a_launch_of_the_feed_forward_block_are_refused(lib):  # noqa: F811
    # 512 threads for 256 rows, 16-bit and narrow: 2^32 threads and more
    most = (1 << 31) - 256
    assert lib.lampa_ff_workspace_bytes(_ff(rows=most, D=8, F=8, x_stride=8), 0) >= 0
    assert lib.lampa_ff_workspace_bytes(_ff(rows=most + 1, D=8, F=8, x_stride=8), 0) == -4
    # 256 threads for a tile of 128 rows x 64 hidden columns
    rows = 128 * ((1 << 24) // 3)
    assert lib.lampa_ff_workspace_bytes(_ff(rows=rows, D=136, F=192, x_stride=136), 0) > 0
    assert lib.lampa_ff_workspace_bytes(_ff(rows=rows, D=136, F=200, x_stride=136), 0) == -4
