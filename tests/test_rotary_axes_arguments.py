"""Arguments of rotary positions of several axes that say something else than what would be turned: refused, not left out."""
import numpy as np
import pytest

from akg_amd import driver, op_desc
from test_attention_ops import builder, refused


def turned(positions, **options):
    b = builder()
    return b.dumps(op_desc.rotary_embedding(b, [b.input([2, 5, 4, 64], "bfloat16")], b.input(positions, "int32"), **options))


def test_sections_are_whole_numbers():
    for sections in ([8.6, 12, 12], [16.5, 16.5], ["16", "16"]):
        with pytest.raises(TypeError):
            turned([len(sections), 5], sections=sections)
    driver.translate(turned([2, 5], sections=np.array([20, 12])))


def test_orders_and_rates_of_axes_need_sections():
    refused(turned([5], axis_order="cycle"), -3, "need sections")
    refused(turned([2, 5], axis_rates="own"), -3, "need sections")
    refused(turned([5], axis_order="rows"), -3, "axis_order")
