"""Times of the sequence operators (genie/sequence.py) on the workloads of perf/operators.py, all in one setting: each pass takes the next of as many input sets as
it needs for 1 GB together, so that nothing a pass reads is left in the last-level cache (256 MB) by the one before.

  python scripts/sequence_kernels.py OUT [NAME ...]

OUT/sequence_operators_kernels.csv: device time of every kernel (rocprofv3 --kernel-trace; the second half of 0.3 s or 2000 passes);  OUT/sequence_operators_calls.csv: time of a call among others, host
included, without the profiler (median of 9 runs of at least 20 ms)."""
import csv
import importlib.util
import os
import statistics
import subprocess
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def operators():
    spec = importlib.util.spec_from_file_location('operators', os.path.join(ROOT, 'perf', 'operators.py'))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.own = True
    return mod


def states(mod, name):
    case = next(c for c in mod.listed() if c['name'] == name)
    n = min(64, max(2, -(-2 ** 30 // max(1, mod.work(case)['bytes']))))
    return [mod.prepare(case, seed) for seed in range(1, n + 1)]


def child_passes(name):
    import torch
    mod = operators()
    sets = states(mod, name)
    end = time.perf_counter() + 0.3
    for i in range(2000):
        mod.run(sets[i % len(sets)])
        if i % 32 == 31:
            torch.cuda.synchronize()
            if time.perf_counter() > end:
                break
    torch.cuda.synchronize()
    print('passes done', name, flush=True)


def child_calls(name):
    import torch
    mod = operators()
    sets = states(mod, name)

    def passes(n):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for i in range(n):
            mod.run(sets[i % len(sets)])
        torch.cuda.synchronize()
        return (time.perf_counter() - t) / n

    passes(2 * len(sets))
    n = max(20, int(0.02 / passes(20)))
    runs = [passes(n) * 1e6 for _ in range(9)]
    print(f'call {statistics.median(runs):.1f} {min(runs):.1f}', flush=True)


def kernel_name(full):
    name = full.replace('void ', '').split('(')[0]
    return name if any(x in name for x in ('packed_', 'cached_', 'decay_')) else None


def main(out, names):
    os.makedirs(out, exist_ok=True)
    out = os.path.abspath(out)
    me, mod = os.path.abspath(__file__), operators()
    env = dict(os.environ, TMPDIR='/tmp')
    kernels, calls = [], []
    for case in mod.listed():
        name = case['name']
        if names and name not in names:
            continue
        r = subprocess.run(['timeout', '-k', '10', '120', sys.executable, me, '--calls', name], cwd=ROOT, env=env, capture_output=True, text=True)
        if r.returncode:
            sys.exit(f'{name}: {r.stdout[-500:]}{r.stderr[-1500:]}')
        _, median, least = next(line for line in r.stdout.splitlines() if line.startswith('call ')).split()
        calls.append([name, median, least])
        d = os.path.join(out, 'trace_' + name)
        r = subprocess.run(['timeout', '-s', 'KILL', '120', 'rocprofv3', '--kernel-trace', '--stats', '-f', 'csv', '-d', d, '-o', 'p', '--', sys.executable, me, '--passes', name],
                           cwd='/tmp', env=env, capture_output=True, text=True)
        if f'passes done {name}' not in r.stdout:
            sys.exit(f'{name}: {r.stdout[-500:]}{r.stderr[-1500:]}')
        seen = {}
        with open(os.path.join(d, 'p_kernel_trace.csv')) as f:
            for row in csv.DictReader(f):
                k = kernel_name(row['Kernel_Name'])
                if k:
                    seen.setdefault((k, row['Grid_Size_X'] + ('' if row['Grid_Size_Y'] == '1' else 'x' + row['Grid_Size_Y'])), []).append(
                        (int(row['End_Timestamp']) - int(row['Start_Timestamp'])) / 1e3)
        for (k, grid), times in seen.items():
            times = times[len(times) // 2:]
            kernels.append([name, k, grid, len(times), f'{statistics.median(times):.1f}', f'{min(times):.1f}'])
        print(f'{name}: call {median} us;', '; '.join(f'{k[1]} {k[4]} ({k[5]})' for k in kernels if k[0] == name), flush=True)
    for path, head, rows in (('kernels', ['workload', 'kernel', 'grid', 'calls', 'median_us', 'min_us'], kernels), ('calls', ['workload', 'median_us', 'min_us'], calls)):
        with open(os.path.join(out, f'sequence_operators_{path}.csv'), 'w', newline='') as f:
            w = csv.writer(f, lineterminator='\n')
            w.writerow(head)
            w.writerows(rows)


if __name__ == '__main__':
    if len(sys.argv) == 3 and sys.argv[1] == '--passes':
        child_passes(sys.argv[2])
    elif len(sys.argv) == 3 and sys.argv[1] == '--calls':
        child_calls(sys.argv[2])
    elif len(sys.argv) >= 2:
        main(sys.argv[1], sys.argv[2:])
    else:
        sys.exit(__doc__)
