"""The e4m3 quantiser where a row has so many blocks that a block's row is found by division in 64 bits."""
import pytest
import torch

from test_fp8_block import DTYPES, F8, bits, blank, laid, margins_untouched, quantize_plain, randn


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("skew", [0, 1])
def test_rows_of_many_blocks(edb, cuda, dtype, skew):
    """9 x 22001 blocks, by wide accesses where the rows are aligned and by single ones where they are not: the same bytes."""
    rows, k = 9, 22000 * 128 + 40
    x = laid(randn(rows, k, seed=8), dtype, skew, skew)
    q, s = blank(rows, k, F8, skew, skew), blank(rows, 22001, torch.float32, 1)
    edb.quantize_fp8(x, q, s)
    want_q, want_s = quantize_plain(x, 1)
    assert torch.equal(bits(q.cpu()), bits(want_q)) and torch.equal(s.cpu(), want_s)
    assert margins_untouched(q) and margins_untouched(s)


@pytest.mark.gpu
def test_wide_accesses_do_not_end_with_the_32_bit_division(edb, cuda):
    """Rows just beyond the last that a 32-bit product divides take no more than twice as long for each: single accesses took
    three times as long.  (k of 6000 blocks: the division changes between 119 and 120 rows.)"""
    k = 6000 * 128
    x = torch.ones(238, k, device="cuda", dtype=torch.bfloat16)
    q, s = torch.empty(238, k, device="cuda", dtype=F8), torch.empty(238, 6000, device="cuda")

    def took(rows):
        times = []
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            edb.quantize_fp8(x[:rows], q[:rows], s[:rows])
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    took(238)
    assert took(238) <= 2 * 2 * took(119)
