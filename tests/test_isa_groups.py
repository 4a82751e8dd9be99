"""CPU-only checks of the generated code of the kernel that goes through shared starts of prompts of many rows: it runs the chunk attention kernel's
loop, with its LDS reads and its matrix instructions in inline assembly, so the same is checked of it."""

from test_isa_hazards import MIN_WAIT_STATES, _kernels, closest_reads, touched_in_flight
from test_isa_operand_reads import _inline_reads_as_transposing


def test_nothing_touches_a_read_in_flight():
    kernels = _kernels("sp_chunk.hip", "sp_groups_kernel")
    assert len(kernels) == 2, "64 / 128 channels"
    for name, body in kernels.items():
        for lines, least in ((_inline_reads_as_transposing(body), 8), (body, 16)):
            count, found = touched_in_flight(lines)
            assert count >= least
            assert not found, f"{name}: '{found[0][1]}' while '{found[0][0]}' is in flight"


def test_no_vector_instruction_reads_an_mfma_result_too_early():
    for name, body in _kernels("sp_chunk.hip", "sp_groups_kernel").items():
        assert sum("v_mfma_f32_16x16x32_bf16" in l for l in body) > 100
        reads = closest_reads(body)
        assert not reads or reads[0][0] >= MIN_WAIT_STATES, (
            f"{name}: '{reads[0][2]}' reads the result of '{reads[0][1]}' only {reads[0][0]} wait states behind it")
