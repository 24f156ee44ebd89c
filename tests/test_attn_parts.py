"""The attention's workspace on the CPU: every part of a sequence begins at 16 bytes, however many rows it has."""
import pytest

import avelang_amd as ave


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("L,Hq", [(1, 1), (3, 1), (1, 5), (1, 2)])
def test_parts_hold_whole_vectors(L, Hq, D):
    # one sequence of 16 units: 16 workgroups, each with a descriptor of 16 bytes and two parts of o, m and the sum
    part = -(-L * Hq * (D + 2) // 4) * 16
    assert ave.paged_attention_workspace_bytes(1, L, Hq, 1, D, 16 * 128) >= 16 * 16 + 16 * 2 * part
