"""Token family: sizes at the edge of what its C entry points take, on the CPU (every call here ends at a check, before a launch)."""
import pytest

P = 1 << 20          # stands for a device address: nothing dereferences it on the host


def embed_bwd(lib, n, D, V, dd, ldd, acc, wb):
    return lib.tad_token_embed_bwd(n, D, V, P, 1, 1.0, P, dd, ldd, P, D, acc, P, wb, None)


@pytest.mark.parametrize("n", [1, 63, 2400, 4096, 5000, 8193, 131073, 1 << 24])
@pytest.mark.parametrize("D", [1, 4, 64, 127, 128, 520, 1000, 4096])
def test_stated_workspace_is_enough_for_every_cut(lib, n, D):
    """A table of 2^30 rows that has to be written whole is refused behind the check of the workspace: with the stated size the
    call gets there whatever the element type and alignment.  Without 16 of its bytes one cut at least does not (of a width that
    packs of four divide: the finest cut is theirs)."""
    need = lib.tad_token_embed_bwd_workspace_bytes(n, D)
    short = 0
    for dd in (0, 1):
        for ldd in (D, D + 1):
            assert embed_bwd(lib, n, D, 1 << 30, dd, ldd, 0, need) == 1
            assert "too many tokens or rows" in lib.tad_last_error().decode()
            assert embed_bwd(lib, n, D, 1 << 30, dd, ldd, 0, need - 16) == 1
            short += "workspace" in lib.tad_last_error().decode()
    assert short > 0 or D % 4 != 0


@pytest.mark.parametrize("n", [1 << 40, 1 << 56, 1 << 58, 1 << 60, 1 << 62, (1 << 63) - 1])
def test_numbers_of_tokens_that_no_memory_holds(lib, n):
    for D in (1, 8, 1000):
        for dtype in (0, 1):
            assert lib.tad_token_embed_fwd(n, D, 5, P, 1, 1.0, P, dtype, D, P, dtype, D, None) == 1
            assert "too many tokens" in lib.tad_last_error().decode()
