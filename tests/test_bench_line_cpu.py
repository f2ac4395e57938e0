"""bench.py's one line holds what was measured without the long series."""

import importlib.util
import json
import os

BENCH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bench.py")


def _bench():
    spec = importlib.util.spec_from_file_location("bench_line", BENCH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_series_are_split_from_the_line():
    mod = _bench()
    configs = {f"C{i}_record": {"us": 1.0 * i, "gbps": 6000.0, "pct_peak": 80.0} for i in range(40)}
    plain = dict(configs)
    for name in mod.SERIES:
        configs[name] = {"points": list(range(1000))}
    rows = [{"N": 2 ** i, "fuselse_us": 1.5 * i, "torch_us": 40.0} for i in range(1, 18)]
    configs["microbench_sweep_512xN_u100"] = {"B": 512, "data": "U(-100,0)", "rows": rows}
    line, series = mod.split_series(configs)
    assert set(series) == set(mod.SERIES) and all(series[k] is configs[k] for k in series)
    assert all(line[k] == v for k, v in plain.items())
    assert line["microbench_sweep_512xN_u100"]["fuselse_us"][1024] == 15.0
    assert set(line) == set(plain) | {"microbench_sweep_512xN_u100"}
    assert len(json.dumps(line)) < 4096
    assert mod.split_series(None) == (None, {})
