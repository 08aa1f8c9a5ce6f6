"""Refusals whose message holds numbers: an error, not the end of the process."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_deformable_refusals_with_numbers(cuda):
    from bevk import load_extension
    ext = load_extension("_modulated_deform_conv_ext")
    x = torch.zeros(1, 8, 6, 5, device=cuda)
    offset, mask = torch.zeros(1, 18, 6, 5, device=cuda), torch.zeros(1, 9, 6, 5, device=cuda)
    packed = ext.dcn_pack_weight(torch.zeros(4, 8, 3, 3, device=cuda), 1)
    with pytest.raises(RuntimeError, match=r"output must be \[1, Cout, 6, 5\]"):
        ext.dcn_forward(x, offset, mask, packed, None, torch.zeros(1, 4, 3, 5, device=cuda),
                        3, 3, 1, 1, 1, 1, 1, 1, 1, 1, False, False)
    columns = torch.zeros(8 * 9 * 30 - 1, device=cuda)
    with pytest.raises(RuntimeError, match="data_col has 2159 elements, expected 2160"):
        ext.modulated_deformable_im2col_cuda(x, offset, mask, 1, 8, 6, 5, 6, 5, 3, 3, 1, 1, 1, 1, 1, 1,
                                             1, columns)
    with pytest.raises(RuntimeError, match="has 2159 elements, expected 2160"):
        ext.dcn_col2im(columns, x, offset, mask, 8, 6, 5, 3, 3, 1, 1, 1, 1, 1, 1, 1,
                       torch.zeros_like(x), None, None)
