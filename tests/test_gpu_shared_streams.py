"""Decode attention of batches whose sequences share pages, from several streams, where the entries' own pages are read by the decode kernels: such
a call has partial results in two workspaces, the one of cut chunks and the one of decode attention."""
import numpy as np
import pytest

from breccia_amd import lib as L
from breccia_amd.kv import DeviceBuffer, Stream, device_sync
from test_gpu_shared import HD, LAYOUTS, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", LAYOUTS)
def test_calls_in_both_workspaces_take_turns(layout):
    with Batch([(2500, [900 + 37 * i for i in range(60)])], layout, n_kv=4, seed=30 + layout) as b:
        n_q, p = 16, b.pool
        p.timing_enable(True)
        qs = [b.queries(n_q) for _ in range(3)]
        want = [b.attend(q) for q in qs]
        # walks, the decode kernels' ranges, the merge: one each a call
        assert [p.timing_read(stage)[0] for stage in (L.STAGE_PREFILL_ATTN, L.STAGE_ATTN_SPLIT, L.STAGE_ATTN_MERGE)] == [3, 3, 3]
        p.timing_enable(False)
        plain = [b.attend(q, plain=True) for q in qs]
        streams = [Stream() for _ in qs]
        qd = [DeviceBuffer.from_numpy(q) for q in qs]
        od, pd = ([DeviceBuffer(q.size * 4) for q in qs] for _ in range(2))
        device_sync()
        for turn in range(12):
            for i in range(3):
                # (the ordinary call writes the decode kernels' workspace as soon as its stream lets it)
                s = streams[(i + turn) % 3]
                p.decode_attn_shared(0, b.seqs, b.pos, b.entries, b.cells, n_q, qd[i], od[i], 1 / 16, stream=s)
                p.decode_attn(0, b.seqs, b.pos, n_q, qd[i], pd[i], 1 / 16, stream=streams[(i + turn + 1) % 3])
            device_sync()
            for i in range(3):
                assert np.array_equal(od[i].download(np.float32).reshape(want[i].shape), want[i]), (turn, i)
                assert np.array_equal(pd[i].download(np.float32).reshape(want[i].shape), plain[i]), (turn, i)
        for x in qd + od + pd:
            x.free()
        for s in streams:
            s.close()
