"""CPU-only checks of the generated code of the chunk attention kernel, whose operands are read by LDS reads in inline assembly as the
short-prompt kernel's are (test_isa_hazards.py, test_isa_operand_reads.py), and whose matrix instructions are inline assembly like the persistent
kernel's."""

from test_isa_hazards import MIN_WAIT_STATES, _kernels, closest_reads, touched_in_flight
from test_isa_operand_reads import _inline_reads_as_transposing


def test_nothing_touches_a_read_in_flight_in_the_chunk_kernel():
    kernels = _kernels("sp_chunk.hip", "sp_chunk_kernel")
    assert len(kernels) == 8, "64 / 128 channels x pages / contiguous x windows / none"
    for name, body in kernels.items():
        for lines, least in ((_inline_reads_as_transposing(body), 8), (body, 16)):
            count, found = touched_in_flight(lines)
            assert count >= least
            assert not found, f"{name}: '{found[0][1]}' while '{found[0][0]}' is in flight"


def test_no_vector_instruction_reads_an_mfma_result_too_early():
    for name, body in _kernels("sp_chunk.hip", "sp_chunk_kernel").items():
        assert sum("v_mfma_f32_16x16x32_bf16" in l for l in body) > 100
        reads = closest_reads(body)
        assert not reads or reads[0][0] >= MIN_WAIT_STATES, (
            f"{name}: '{reads[0][2]}' reads the result of '{reads[0][1]}' only {reads[0][0]} wait states behind it")


def test_nothing_touches_a_read_in_flight_in_the_single_token_kernel():
    kernels = _kernels("sp_paged_decode.hip", "sp_paged_decode_kernel")
    assert len(kernels) == 4, "64 / 128 channels x pages / contiguous"
    for name, body in kernels.items():
        for lines, least in ((_inline_reads_as_transposing(body), 4), (body, 8)):
            count, found = touched_in_flight(lines)
            assert count >= least
            assert not found, f"{name}: '{found[0][1]}' while '{found[0][0]}' is in flight"
