"""What moe_fp8_layer_workspace_bytes asks for: host code only."""
import pytest

import moe_prefetch

L = moe_prefetch.lib()


def up256(n):
    return -(-n // 256) * 256


@pytest.mark.parametrize("T, E, K, H, I", [(2048, 128, 8, 2048, 768), (1000, 64, 8, 2048, 512), (513, 256, 1, 300, 1000), (8191, 256, 8, 7168, 2048),
                                           (65, 128, 8, 2048, 768)])
def test_a_dispatch_keeps_h_and_the_rows_in_one_place(T, E, K, H, I):
    # codes and scales of x and h, the dispatch's lists, and f32 for the longer of h and a row for each pair
    P = T * K
    codes = sum(up256(n * (-(-k // 16) * 16)) + up256(n * (-(-k // 128)) * 4) for n, k in ((T, H), (P, I)))
    lists = up256(E * 4) + up256((E + 1) * 4) + up256(P * 4)
    assert L.moe_fp8_layer_workspace_bytes(T, E, K, H, I) == codes + lists + up256(P * max(H, I) * 4)


@pytest.mark.parametrize("T, E, K, H, I", [(64, 128, 8, 2048, 768), (1, 8, 2, 256, 128), (512, 16, 1, 128, 512)])
def test_few_pairs_keep_both(T, E, K, H, I):
    assert L.moe_fp8_layer_workspace_bytes(T, E, K, H, I) >= T * K * (H + I) * 4
