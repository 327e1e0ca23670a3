"""A step plan of an e4m3 pool tells exactly where it is: while it has cells left, at its last one, and when it is asked to go past it."""
import numpy as np
import pytest

import f8p_model as M
from breccia_amd.kv import DeviceBuffer, Graph, StepPlan, Stream
from test_gpu_f8p import fill, rng_of, rows_of

pytestmark = pytest.mark.gpu


def test_state_of_a_plan_up_to_its_horizon_and_past_it():
    lens, n_q, horizon = [31, 200, 16], 16, 5
    with M.F8Twin(n_pages=64) as tw:
        seqs = [tw.pool.seq_create() for _ in lens]
        for s, n in zip(seqs, lens):
            fill(tw, s, n, rng_of(70, s))
            tw.pool.seq_reserve(s, n + horizon)
        rng, st = rng_of(71), Stream()
        x = rows_of(rng, len(lens), 2)
        kd, vd = DeviceBuffer.from_numpy(x), DeviceBuffer.from_numpy(x)
        qd = DeviceBuffer.from_numpy(rng.standard_normal((len(lens), n_q, 256)).astype(np.float32))
        od = DeviceBuffer(len(lens) * n_q * 1024)
        plan = StepPlan(tw.pool, seqs, lens, horizon, n_q, st)
        st.sync()
        graph = Graph(st)
        plan.decode(0, kd, vd, qd, od, 1 / 16.0, stream=st)
        plan.advance(st)
        graph.end()
        for t in range(horizon + 2):
            pos, steps, status = plan.state(st)
            done = min(t, horizon - 1)                      # the last cell is where it stays
            assert pos.tolist() == [n + done for n in lens] and steps == done and status == int(t >= horizon), t
            if t < horizon:
                for s, n, row in zip(seqs, lens, x):
                    assert tw.images[0].append(tw.pool.block_table(s), n + t, row[None], row[None]) == 0
            graph.launch()
        st.sync()
        tw.assert_pools_equal()                             # asked again past the horizon, it writes the last cell again
        graph.destroy()
        plan.destroy()
