"""Page tables on the GPU: calls from several host threads, and shortages past 32 bits."""
from __future__ import annotations

import threading

import pytest
import torch

from wal2026_b200.kv8 import kv_pages_assign

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_assign_from_threads_with_different_row_counts():
    # calls whose shared memory differs, at the same time: none may take away what another needs
    errors = []

    def work(rows):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                table, zero, one = _i32([[0, 1]]), torch.zeros(rows, dtype=torch.int32, device=DEV), None
                one = torch.ones_like(zero)
                out = torch.empty(rows, 2, dtype=torch.int32, device=DEV)
                ref, src, dst = (torch.empty(n, dtype=torch.int32, device=DEV) for n in (rows + 8, rows, rows))
                info = torch.empty(2, dtype=torch.int32, device=DEV)
                for _ in range(400):
                    kv_pages_assign(table, zero, zero, one, 16, out, ref, src, dst, info)
                torch.cuda.current_stream().synchronize()
                assert info.tolist() == [8, 0] and out[:, 0].tolist() == list(range(rows))
        except Exception as e:  # noqa: BLE001 - handed to the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in (3600, 16000, 4200, 9000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("rows,add", [(16, 2 ** 31 - 1), (32, 2 ** 31 - 1), (3, 2 ** 31 - 1), (40, 1 << 20)])
def test_assign_counts_shortages_past_32_bits(rows, add):
    # the pages that rows ask for beyond their width, summed: 2^27 each, kept within an int32
    P, width, pages = 16, 2, 5
    table = torch.full((1, width), -1, dtype=torch.int32, device=DEV)
    out, ref = torch.empty(rows, width, dtype=torch.int32, device=DEV), torch.empty(pages, dtype=torch.int32, device=DEV)
    src, dst, info = (torch.empty(n, dtype=torch.int32, device=DEV) for n in (rows, rows, 2))
    kv_pages_assign(table, _i32([-1] * rows), _i32([0] * rows), _i32([add] * rows), P, out, ref, src, dst, info)
    want = rows * -(-add // P) - pages
    assert info.tolist() == [0, min(want, 2 ** 31 - 1)]
