"""GPU tests of prefix pages that are not in the pool: they read as rows of zeros, whatever their number."""
import pytest
import torch

from test_shared_prefix_gpu import check, problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api():
    import decoding_attention_b200
    return decoding_attention_b200


@pytest.mark.parametrize("bad", [-1, 1 << 20, 1 << 25, 1 << 26, (1 << 26) + 1, 1 << 28, 1 << 30, 2 ** 31 - 1, -2 ** 31, -(1 << 26)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_pages_outside_the_pool_in_full_tiles_and_in_the_last(api, page, bad):
    prefix = 600  # four full tiles and one of 88 keys
    for one_pool in (False, True):
        pr = problem(torch.bfloat16, prefix, [10, 0, 20], 8, 2, 128, 40, page=page, prefix_page=page, one_pool=one_pool)
        blocks = len(pr["args"]["prefix_table"])
        for i in (0, blocks // 2, blocks - 1):
            pr["args"]["prefix_table"][i] = bad
            for side in pr["keys"]:
                for x in side:
                    x[i * page:min(prefix, (i + 1) * page)] = 0
        check(api, pr, what=f"page {page}, entry {bad}")
