"""Instructions that every lane of a warp has to reach together (`.aligned`), read in the sources.

After a branch that only some lanes take, the hardware may run the lanes of a warp apart; an aligned
instruction reached that way is undefined, and an aligned barrier may then never complete.
"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / 'redshift_b200' / 'csrc'


def _function(text, name):
    start = re.search(r'void ' + name + r'\([^)]*\) \{', text).end()
    return text[start:text.index('\n}', start)]


@pytest.mark.parametrize('source,name', [('mm8.cu', 'cluster_sync')])
def test_a_warp_meets_in_front_of_a_barrier(source, name):
    body = _function((CSRC / source).read_text(), name)
    assert '__syncwarp();' in body and body.index('__syncwarp();') < body.index('asm volatile')
