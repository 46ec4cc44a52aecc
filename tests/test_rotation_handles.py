"""What a Rotation hands to the library stays what it was built with (no GPU): copies,
pickles and attributes of a rotation."""

from __future__ import annotations

import copy
import ctypes
import gc
import pickle

import numpy as np
import pytest

import paged


def handed_over(r):
    """(frequencies, axes) at the addresses that a call hands to the library."""
    freq, axis, pairs, _ = r._args
    return ((ctypes.c_double * pairs).from_address(freq)[:],
            list((ctypes.c_uint8 * pairs).from_address(axis)))


def rotations():
    return [paged.Rotation(8, 100.0), paged.Rotation(12, 50.0, [1, 2, 3], order="ladders", neox=False),
            paged.Rotation(16, 100.0, [4, 2, 2], order="cyclic"),
            paged.Rotation(6, inv_freq=[1.0, 0.5, -0.25])]


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda r: copy.deepcopy({"rope": [r]})["rope"][0],
                                 lambda r: pickle.loads(pickle.dumps(r))],
                         ids=["copy", "deepcopy", "deepcopy-in-a-config", "pickle"])
def test_a_copy_hands_over_its_own_tables(how):
    for i in range(len(rotations())):
        r = rotations()[i]
        want = (r.inv_freq.tolist(), r.axis.tolist())
        rest = (r.rotary_dim, r.pairs, r.axes, r.neox)
        c = how(r)
        # every address a copy hands over is that of an array that it keeps
        assert c._args[:2] == (c.inv_freq.ctypes.data, c.axis.ctypes.data)
        del r
        gc.collect()
        filler = [np.full(n, 7.0) for n in (3, 4, 6, 8) for _ in range(64)]
        assert handed_over(c) == want and (c.inv_freq.tolist(), c.axis.tolist()) == want
        assert (c.rotary_dim, c.pairs, c.axes, c.neox) == rest and c._args[2:] == (rest[1], int(rest[3]))
        assert len(filler) == 256


@pytest.mark.parametrize("name", ["inv_freq", "axis", "rotary_dim", "pairs", "axes", "neox", "_args"])
def test_a_rotation_does_not_change(name):
    """A new value would leave calls with the addresses of the old tables."""
    r = paged.Rotation(8, 100.0)
    want = handed_over(r)
    with pytest.raises(AttributeError):
        setattr(r, name, getattr(r, name))
    with pytest.raises(AttributeError):
        delattr(r, name)
    assert handed_over(r) == want == (r.inv_freq.tolist(), r.axis.tolist())
    for table in (r.inv_freq, r.axis):
        with pytest.raises(ValueError):
            table[0] = 3


def test_what_a_program_adds_to_a_rotation_goes_along():
    class Named(paged.Rotation):
        pass
    r = Named(8, 100.0)
    r.label = ["long"]
    for c in (copy.copy(r), copy.deepcopy(r)):
        assert type(c) is Named and c.label == ["long"] and handed_over(c) == handed_over(r)
    del r.label
    assert not hasattr(r, "label")
