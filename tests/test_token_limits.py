"""Token family: sizes at the edge of what its C entry points take, on the CPU (every call here ends at a check, before a launch)."""
import pytest

P = 1 << 20          # stands for a device address: nothing dereferences it on the host


def embed_bwd(lib, n, D, V, dd, ldd, acc, wb):
    return lib.tad_token_embed_bwd(n, D, V, P, 1, 1.0, P, dd, ldd, P, D, acc, P, wb, None)


@pytest.mark.parametrize("n", [1 << 40, 1 << 56, 1 << 58, 1 << 60, 1 << 62, (1 << 63) - 1])
def test_numbers_of_tokens_that_no_memory_holds(lib, n):
    for D in (1, 8, 1000):
        for dtype in (0, 1):
            assert lib.tad_token_embed_fwd(n, D, 5, P, 1, 1.0, P, dtype, D, P, dtype, D, None) == 1
            assert "too many tokens" in lib.tad_last_error().decode()
