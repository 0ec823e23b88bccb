"""CPU test of the built library: of the row norms' kernels it holds those that some size reaches, and no other."""
import re

from helpers import ROOT

LIBRARY = ROOT / "minicpm-v-4.6-orangepi_amd" / "lib" / "libmcv_quant.so"


def test_row_norms():
    names = set(re.findall(rb"_ZN3mcv14rms_row_kernelILi(\d+)ELb(\d)ELb(\d)ELb(\d)E", LIBRARY.read_bytes()))
    have = {tuple(int(x) for x in n) for n in names}             # elements a thread, in chunks, to int8, of a sum
    per = [(0, 0), (1, 0)] + [(n, vec) for n in (4, 8, 16, 32) for vec in (0, 1)]
    want = {(n, vec, quant, add) for n, vec in per for quant in (0, 1) for add in (0, 1)}
    assert have == {k for k in want if not (k[0] == 1 and k[3])}     # sums of up to 256 have a wave a row
