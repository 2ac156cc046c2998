"""What the functions around the operator refuse at the ends of what they take: without a GPU, before anything is launched."""
import ctypes

ONE, NULL = ctypes.c_void_p(256), ctypes.c_void_p(0)          # never dereferenced: the checks come first


def test_a_table_gradient_of_too_many_places():
    """The batch elements of a place that one float would add up: as many as a table's gradient takes at a time, or places of their own."""
    from dfa3D import _lib
    lib = _lib.lib()
    for R, N in ((2 ** 20 + 1, 2 ** 10), (2 ** 31, 1), (2 ** 30 + 1, 1)):
        assert lib.dfa3d_embedding_grad_table_workspace_bytes(R, N, 7, 2, 8, 0) == 0 and b"2^30" in lib.dfa3d_last_error()
        assert lib.dfa3d_embedding_grad_table(NULL, ONE, 4, NULL, ONE, ONE, NULL, ONE, 1 << 40, R, N, 7, 2, 8, 1.0, 0, NULL) == -2 and b"2^30" in lib.dfa3d_last_error()
    for R, N in ((2 ** 20, 2 ** 11), (2 ** 30, 1), (2 ** 20 + 1, 1000), (1, 2 ** 30)):
        assert lib.dfa3d_embedding_grad_table_workspace_bytes(R, N, 7, 2, 8, 0) > 0


def test_batch_elements_are_places_of_their_own():
    """Which the workspace shows: that of R N places of one batch element, or that of N."""
    from dfa3D import _lib
    need = _lib.lib().dfa3d_embedding_grad_table_workspace_bytes
    for R, N, V, H, E in ((10000, 100, 100, 1, 256), (20000, 100, 100, 1, 256), (2 ** 25, 1, 1, 1, 8), (2 ** 21, 1, 9, 512, 512), (2 ** 30, 1, 1, 1, 1)):
        assert need(R, N, V, H, E, 0) == need(1, R * N, V, H, E, 0)
    for R, N, V, H, E in ((7, 200000, 1, 1, 256), (16, 2 ** 20, 2 ** 19, 1, 256), (64, 2000, 2000, 8, 256)):
        assert need(R, N, V, H, E, 0) == need(1, N, V, H, E, 0)


def test_a_norm_of_too_many_levels():
    """Of all batch elements together, whose channels' sums are numbered in 31 bits."""
    from dfa3D import _lib
    lib = _lib.lib()
    size = lib.dfa3d_group_norm_workspace_bytes
    assert size(2 ** 26 + 1, 1, 8, 2, 16, 1, 0) == 0 and b"2^30 levels" in lib.dfa3d_last_error()
    assert size(2 ** 30, 1, 8, 2, 1, 0, 0) > 0
    assert lib.dfa3d_group_norm(ONE, NULL, NULL, ONE, ONE, ONE, ONE, 1 << 50, 2 ** 26 + 1, 1, 8, 2, 16, 1e-5, 0, 0, NULL) == -2
