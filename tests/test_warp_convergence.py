"""Instructions that every lane of a warp has to reach together (`.aligned`), read in the sources.

After a branch that only some lanes take, the hardware may run the lanes of a warp apart; an aligned
instruction reached that way is undefined, and an aligned barrier may then never complete.
"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / 'redshift_b200' / 'csrc'
# a branch on the lane or the thread, or on a value that each lane has for itself
SPLITS = re.compile(r'if \([^)]*(\blane\b|threadIdx\.x == 0|m_use\[u\]|\brow4?\b|\bcol\b)')
MEETS = re.compile(r'__syncwarp|__syncthreads|_wait8?\(|__shfl|__any_sync|__all_sync|named_barrier|cluster_sync|__reduce_max_sync')
TOGETHER = re.compile(r'\btmem_(ld|st)\w*\(')


def _function(text, name):
    start = re.search(r'void ' + name + r'\([^)]*\) \{', text).end()
    return text[start:text.index('\n}', start)]


@pytest.mark.parametrize('source,name', [('common.cuh', 'named_barrier'), ('mm8.cu', 'cluster_sync')])
def test_a_warp_meets_in_front_of_a_barrier(source, name):
    body = _function((CSRC / source).read_text(), name)
    assert '__syncwarp();' in body and body.index('__syncwarp();') < body.index('asm volatile')


@pytest.mark.parametrize('source', ['attention8.cu', 'mm8.cu'])
def test_a_warp_meets_in_front_of_an_access_to_tensor_memory(source):
    split, apart = None, []
    for number, line in enumerate((CSRC / source).read_text().split('\n'), 1):
        code = line.split('//')[0]
        if TOGETHER.search(code) and split:
            apart.append((split, number))
        if MEETS.search(code):
            split = None
        elif SPLITS.search(code) and 'lane < 16' not in code:
            split = number
    assert not apart, apart
