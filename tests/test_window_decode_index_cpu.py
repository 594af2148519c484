"""The single-token form's position arithmetic in 32-bit integers, restated: at
every length an int holds, no intermediate leaves the type and no slot the
cache."""

import pytest

LAST = 2**31 - 1


def _int(v):
    assert -2**31 <= v <= LAST, "leaves 32 bits"
    return v


def _view(n, window, sinks, capacity):
    """(sinks seen, first ring slot, positions) as window_decode_kernel forms them."""
    ring = _int(capacity - sinks)
    sink = 0 if n < 0 else _int(n + 1) if n < sinks else sinks
    lo = max(sinks, _int(_int(n - window) + 1))
    cnt = 0 if n < 0 else _int(sink + (0 if n < lo else _int(_int(n - lo) + 1)))
    first = _int(lo - sinks) % ring if lo > sinks else 0
    return sink, first, cnt


@pytest.mark.parametrize("window,sinks,slack", [(1, 0, 0), (1, 4, 0), (16, 4, 0), (16, 0, 3), (64, 130, 0), (8192, 16, 0)])
def test_positions_at_every_length(window, sinks, slack):
    cap = sinks + window + slack
    for n in list(range(-2, 3 * window + sinks + 3)) + [2**30, LAST - 1, LAST]:
        sink, first, cnt = _view(n, window, sinks, cap)
        seen = set(range(min(sinks, n + 1))) | set(range(max(0, n + 1 - window), n + 1)) if n >= 0 else set()
        assert cnt == len(seen)
        for pos, at in ((n, cnt - 1), (max(sinks, n + 1 - window), sink)):  # the new token, the window's first
            if n >= sinks:
                slot = first + at - sink
                slot = sinks + (slot - (cap - sinks) if slot >= cap - sinks else slot)
                assert slot == sinks + (pos - sinks) % (cap - sinks) and sinks <= slot < cap
