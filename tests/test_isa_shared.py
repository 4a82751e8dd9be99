"""CPU-only check of the generated code of the kernel for shared starts of prompts, whose operands are read by LDS reads in inline assembly as the
single-token kernel's are: nothing may touch a read's registers, and no branch or label stand, between the read and the wait that covers it."""

from test_isa_hazards import _kernels, touched_in_flight
from test_isa_operand_reads import _inline_reads_as_transposing


def test_nothing_touches_a_read_in_flight():
    kernels = _kernels("sp_shared_prefix.hip", "sp_shared_kernel")
    assert len(kernels) == 2, "64 / 128 channels"
    for name, body in kernels.items():
        for lines, least in ((_inline_reads_as_transposing(body), 8), (body, 16)):
            count, found = touched_in_flight(lines)
            assert count >= least
            assert not found, f"{name}: '{found[0][1]}' while '{found[0][0]}' is in flight"


def test_the_loops_keep_their_registers():
    """What the kernel sets aside in memory is set aside outside the loops over the keys."""
    for name, body in _kernels("sp_shared_prefix.hip", "sp_shared_kernel").items():
        products = [i for i, l in enumerate(body) if "v_mfma" in l]
        runs = [[products[0], products[0]]]
        for i in products:
            if i - runs[-1][1] > 400:  # the two loops
                runs.append([i, i])
            runs[-1][1] = i
        for a, b in runs:
            assert not [l for l in body[a:b] if "scratch_" in l], name
