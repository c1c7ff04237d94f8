"""Linear attention's gradient takes the heads of a group in turn all of them or not at all: the workspace says which (CPU), and sizes
at which only a part of a group would leave enough workgroups are right under the bounds of test_gpu_attention.py (GPU)."""
import pytest
import torch

from boa_amd import _native
from test_gpu_attention import BF, F16, F32, _check
from test_more_ops_args import _packed

SIZES = [(300, 65, 8, 1, 16, 8), (150, 65, 12, 1, 9, 70), (100, 300, 6, 1, 20, 5), (40, 1000, 16, 2, 64, 64), (600, 65, 4, 1, 9, 9), (1, 64, 8, 1, 8, 8)]


@pytest.mark.parametrize("n,length,heads,groups,key,value", SIZES)
def test_all_heads_of_a_group_or_one(n, length, heads, groups, key, value):
    lib = _native.load_cdll()
    need = lambda g: lib.boa_linear_attention_work_bytes(_packed(n=n, length=length, heads=heads, groups=g, key=key, value=value), 1)  # noqa: E731
    tiles = -(-value // 64)

    def sums(g, parts):  # dq's and dk's parts in float32, where there are several
        return 2 * 4 * n * length * g * key * parts if parts > 1 else 0

    own = need(heads) - sums(heads, tiles)  # what does not hang on the groups
    assert need(groups) - own in (sums(groups, tiles), sums(groups, heads // groups * tiles))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("size,decay", [(SIZES[0], "token"), (SIZES[1], "head"), (SIZES[2], "token")])
def test_gradients_where_a_part_of_a_group_would_do(gpu, size, decay, dtype):
    _check(*size, dtype, decay, ragged=True, state=True, seed=3)
