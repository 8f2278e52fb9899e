"""The bits of the device error word: one for each kind of wait, so that a report tells which one gave up."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tiny-kernel_b200", "csrc")


def test_every_wait_has_a_bit_of_its_own():
    bits = {}
    for path in sorted(glob.glob(os.path.join(CSRC, "*"))):
        with open(path) as f:
            for name, value in re.findall(r"constexpr unsigned (kErr\w+) = (\d+)u;", f.read()):
                if name != "kErrHostSlots":  # a number of slots
                    bits[name, os.path.basename(path)] = int(value)
    assert len(bits) >= 7 and all(v & v - 1 == 0 for v in bits.values())
    assert len(set(bits.values())) == len(bits), bits
