"""The hand-over of a split row's list (vqa_sample, few long rows): every wave of a workgroup stores its share of the list, and one
thread then says that the workgroup is done.  Its release waits for its own wave's stores only, and a barrier waits for no
store at all: each wave has to wait for its own before the barrier.  Seen in the compiler's output; needs no GPU."""
import os
import subprocess

import pytest

from vqa_amd import build


@pytest.fixture(scope='module')
def assembly(tmp_path_factory):
    if not os.path.exists(build.HIPCC):
        pytest.skip('no compiler')
    out = str(tmp_path_factory.mktemp('asm') / 'sample.s')
    subprocess.check_call([build.HIPCC] + build.FLAGS + ['--offload-device-only', '-S', os.path.join(build.CSRC, 'sample.hip'), '-o', out],
                          stderr=subprocess.DEVNULL)
    with open(out) as f:
        return [line.split(';')[0].strip() for line in f]


def test_every_wave_waits_for_its_stores_before_the_barrier(assembly):
    releases = [i for i, line in enumerate(assembly) if line.startswith('buffer_wbl2')]
    assert len(releases) == 3                                  # one for each type of logits
    for r in releases:
        barrier = max(i for i in range(r) if assembly[i] == 's_barrier')
        store = max(i for i in range(barrier) if assembly[i].startswith('global_store') and assembly[i].endswith('sc1'))
        label = max(i for i in range(barrier) if assembly[i].endswith(':'))
        assert store < label                                   # the block that ends in the barrier: every wave comes through it
        assert 's_waitcnt vmcnt(0)' in assembly[label:barrier], '\n'.join(assembly[store:r + 1])
