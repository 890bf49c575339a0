"""CPU: attn_cross_kernel is built in the forms that its planner takes, no others."""
import re

from test_kernel_resources import kernels


def test_cross_kernels_are_those_of_the_planner(tmp_path):
    """plan_cross: 4 waves at every head_dim, 8 at 32 and 128."""
    built = {tuple(map(int, m.groups())) for name in kernels("attention_cross.o", tmp_path)
             if (m := re.search(r"attn_cross_kernelILi(\d+)ELb[01]ELi(\d)E", name))}
    assert built == {(32, 4), (32, 8), (64, 4), (128, 4), (128, 8), (256, 4)}
