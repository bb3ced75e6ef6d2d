cd $GRAFT_REPO_ROOT
mkdir -p gpurun_out/r03_b
export PYTHONUNBUFFERED=1
timeout 1500 python -m pytest tests/test_side_stream.py tests/test_trainer_glue.py tests/test_gpu_parity.py tests/test_full_size.py -m gpu -q -s 2>&1 | tail -80 > gpurun_out/r03_b/tests.txt
SWEEP_POISON=1 SWEEP_REPEAT=2 timeout 900 python -u tests/sweep_layers.py 80 1 2>&1 | tail -20 > gpurun_out/r03_b/sweep_layers_1.txt
tail -n 5 gpurun_out/r03_b/tests.txt gpurun_out/r03_b/sweep_layers_1.txt
