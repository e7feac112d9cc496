"""Bytes that an input gradient asks for, by its number of tokens."""
from diffuser_b200 import _lib


def test_no_workspace_where_one_launch_decodes_and_multiplies():
    lib = _lib.lib()
    whole = 4096 * 1024 * 2
    assert lib.dq_linear_dgrad_workspace(4096, 1024) == whole
    for m, n, nbytes in ((0, 4096, 0), (1, 4096, 0), (256, 4096, 0), (512, 4096, 0), (513, 4096, whole),
                         (256, 1024, 0), (257, 1024, whole // 4), (512, 2048, 0), (512, 2040, 2040 * 2048),
                         (6144, 4096, whole)):
        assert lib.dq_linear_dgrad_workspace_for(m, n, 1024) == nbytes, (m, n)
    assert lib.dq_linear_dgrad_workspace_for(600, 0, 1024) == 0
