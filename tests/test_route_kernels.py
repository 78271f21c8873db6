"""The library holds the routing kernels that a call can reach, and no others: the names in its own code objects."""
import re

from test_resident_blocks import PKG, device_objects


def test_no_kernel_without_a_call():
    lib = (PKG / "build" / "libpaia_gemv.so").read_bytes()
    found = {m for elf in device_objects(lib)
             for m in re.findall(rb"route_kernelILi(\d+)ELb([01])ELb([01])ELb([01])E\w*\.kd", elf)}
    one = (b"0", b"1")
    choosing = {(n, sigmoid, b"1", alone) for n in (b"1", b"2", b"4", b"8", b"16") for sigmoid in one for alone in one}
    given = {(b"1", b"0", b"0", alone) for alone in one}           # ids that the caller has: no logits to hold
    assert found == choosing | given
