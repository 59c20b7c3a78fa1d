"""Which work a call of a context waits for on the GPU, when streams change and some are captured into graphs between: vq_b200/csrc/stream_order.hpp over a
model of streams and one event, on the CPU."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_every_call_is_behind_the_work_of_those_before_it(tmp_path):
    exe = os.path.join(str(tmp_path), "test_stream_order")
    subprocess.check_call(["/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-o", exe, os.path.join(HERE, "cpp", "test_stream_order.cpp")])
    res = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=300)
    out = res.stdout.decode()
    assert res.returncode == 0 and "all checks of the order of calls passed" in out, out[:3000]
