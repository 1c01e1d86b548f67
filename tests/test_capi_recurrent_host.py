"""Host-side checks of the gated recurrence's and the feed-forward block's C entry points: sizes, and what they refuse before any
launch. No kernel is launched here."""
import os

import pytest

from lampa_amd import _capi
from lampa_amd import feed_forward as ff
from lampa_amd import linear_recurrence as lr

LR = dict(zip(("x decay_gate input_gate gate A h0 y ht tile_states cu dy dht dx ddecay dinput dgate dA dh0 workspace workspace_bytes n_tokens "
               "seq_len x_stride decay_stride input_stride gate_stride n_seq D dtype activation normalize reserved").split(), range(32)))
FF = dict(zip("x w_gate w_up w_down y dy dx dw_gate dw_up dw_down workspace workspace_bytes rows x_stride D F dtype activation".split(),
              range(18)))
FAKE = 1 << 20  # an aligned address that nothing reads: every call here is refused first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_capi.LIB_PATH):
        from lampa_amd import build

        build.build(verbose=False)
    return _capi.lib()


def _lr(**kw):
    v = [0] * 32
    base = dict(x=FAKE, decay_gate=FAKE, A=FAKE, y=FAKE, n_tokens=1000, seq_len=1000, x_stride=512, decay_stride=512, n_seq=1, D=512,
                normalize=1)
    for k, x in {**base, **kw}.items():
        v[LR[k]] = x
    return lr._ARGS.pack(*v)


def _ff(**kw):
    v = [0] * 18
    base = dict(x=FAKE, w_gate=FAKE, w_up=FAKE, w_down=FAKE, y=FAKE, rows=100, x_stride=128, D=128, F=512)
    for k, x in {**base, **kw}.items():
        v[FF[k]] = x
    return ff._ARGS.pack(*v)


def test_tiles_and_words_of_the_recurrence(lib):
    # 512 channels: 64 lanes of two side by side, tiles of 64 tokens
    assert lib.lampa_lr_slots(_lr()) == 16
    assert lib.lampa_lr_slots(_lr(cu=FAKE, n_seq=5)) == 1000 // 64 + 6
    assert lib.lampa_lr_slots(_lr(n_tokens=0, seq_len=0, n_seq=3)) == 3
    assert lib.lampa_lr_slots(_lr(D=24, x_stride=24, decay_stride=24)) == 4   # tiles of 256
    words = lib.lampa_lr_workspace_bytes(_lr(), 0)
    assert words >= 16 * 512 * 8 and lib.lampa_lr_workspace_bytes(_lr(), 1) >= words + 16 * 512 * 4
    assert lib.lampa_lr_workspace_bytes(_lr(n_tokens=64, seq_len=64), 0) < 1024  # one tile: nothing to hand on


def test_refusals_of_the_recurrence(lib):
    for code, kw in ((-1, dict(D=0)), (-1, dict(dtype=3)), (-1, dict(activation=3)), (-1, dict(n_seq=0)), (-1, dict(seq_len=999)),
                     (-1, dict(seq_len=2000, n_tokens=1000)), (-4, dict(D=(1 << 20) + 1))):
        assert lib.lampa_lr_slots(_lr(**kw)) == code, kw
    size = lib.lampa_lr_workspace_bytes(_lr(), 0)
    ok = dict(workspace=FAKE, workspace_bytes=size)
    for code, kw in ((-1, dict(ok, x=0)), (-1, dict(ok, A=0)), (-1, dict(ok, y=0)), (-1, dict(ok, x_stride=511)),
                     (-4, dict(ok, x_stride=1 << 24)), (-2, dict(workspace=FAKE, workspace_bytes=size - 1)), (-2, dict()),
                     (-1, dict(ok, workspace=FAKE + 4))):
        assert lib.lampa_lr_scan_fwd(_lr(**kw), None) == code, kw
    back = dict(workspace=FAKE, workspace_bytes=1 << 40, dy=FAKE, dx=FAKE, ddecay=FAKE, dA=FAKE, tile_states=FAKE)
    for kw in (dict(back, dA=0), dict(back, tile_states=0), dict(back, dx=0), dict(back, h0=FAKE), dict(back, gate=FAKE, gate_stride=512),
               dict(back, input_gate=FAKE, input_stride=512)):
        assert lib.lampa_lr_scan_bwd(_lr(**kw), None) == -1, kw
    step = lambda **kw: lib.lampa_lr_step(*[{**dict(x=FAKE, xs=8, r=FAKE, rs=8, i=0, is_=0, z=0, zs=0, A=FAKE, s=FAKE, n=FAKE, y=FAKE,  # noqa: E731
                                                   rows=2, D=8, dt=0, act=0, norm=1, stream=None), **kw}[k]
                                            for k in ("x", "xs", "r", "rs", "i", "is_", "z", "zs", "A", "s", "n", "y", "rows", "D", "dt", "act", "norm", "stream")])
    assert step(x=None) == -1 and step(xs=7) == -1 and step(dt=3) == -1 and step(act=5) == -1 and step(D=0) == -1
    assert step(i=FAKE, is_=4) == -1 and step(rows=0) == 0


def test_workspaces_and_refusals_of_the_feed_forward_block(lib):
    assert lib.lampa_ff_workspace_bytes(_ff(rows=60000), 0) == 0                      # hidden values stay in registers
    assert lib.lampa_ff_workspace_bytes(_ff(rows=60000, dtype=2), 0) >= 60000 * 512 * 4
    assert lib.lampa_ff_workspace_bytes(_ff(rows=60000), 1) >= 3 * 128 * 512 * 4
    for code, kw in ((-1, dict(D=0)), (-1, dict(F=0)), (-1, dict(dtype=3)), (-1, dict(activation=-1)), (-4, dict(D=12)), (-4, dict(F=20)),
                     (-4, dict(D=1 << 18)), (-1, dict(rows=-1))):
        assert lib.lampa_ff_workspace_bytes(_ff(**kw), 0) == code, kw
    ok = dict(workspace=FAKE, workspace_bytes=1 << 40)
    for code, kw in ((-1, dict(ok, x=0)), (-1, dict(ok, w_up=0)), (-1, dict(ok, y=0)), (-1, dict(ok, x=FAKE + 8)), (-1, dict(ok, x_stride=64)),
                     (-4, dict(ok, x_stride=132)), (-4, dict(ok, x_stride=1 << 21)), (-2, dict())):
        assert lib.lampa_ff_fwd(_ff(**kw), None) == code, kw
    assert lib.lampa_ff_fwd(_ff(**ok, rows=0), None) == 0
    assert lib.lampa_ff_bwd(_ff(**ok, dx=FAKE), None) == -1                            # no dy
    assert lib.lampa_ff_bwd(_ff(**ok, dy=FAKE), None) == 0                             # nothing asked for
