# Top-level build.  Everything is built in-tree so the artefacts travel with the
# snapshot to the GPU box (they are git-ignored, not gpurun-ignored).
#
#   make lib      libnvk_paged_attn.so: HIP kernels + C ABI, gfx950 only
#   make cli      nano_vllm_amd/nvk_run: the reference's command line over the library
#   make oracle   the CPU checker (oracle/, test infrastructure)
#   make ref      the reference's own headers behind a shim (only where /root/reference exists)
#   make all      all of the above

HIPCC   ?= /opt/rocm/bin/hipcc
ARCH    ?= gfx950
CSRC    := nano_vllm_amd/csrc
LIB     := nano_vllm_amd/libnvk_paged_attn.so
# No packed fp32 instructions (v_pk_add / mul / fma_f32): some of their forms have given wrong results on this machine.
# (A device feature: hipcc's host pass says that it does not know it, which is harmless.)
HIPFLAGS := --offload-arch=$(ARCH) -O3 -std=c++17 -fPIC -Iinclude -I$(CSRC) -Wall -Wno-unused-function -fno-gpu-rdc \
            -Xclang -target-feature -Xclang -packed-fp32-ops $(EXTRA)
EXTRA    ?=
OBJ      := build/obj
HIP_SRC  := nvk_paged_attn nvk_batch nvk_linear nvk_model nvk_shard nvk_rotary nvk_mx4 nvk_sparse
CPP_SRC  := nvk_block_manager nvk_tokenizer nvk_model_group
OBJS     := $(HIP_SRC:%=$(OBJ)/%.o) $(CPP_SRC:%=$(OBJ)/%.o)
HEADERS  := $(wildcard $(CSRC)/*.h) include/nvk_paged_attn.h

.PHONY: all lib cli oracle ref clean asm asan
all: lib cli oracle ref

lib: $(LIB)

# one object per source (make -j builds them side by side; without -fgpu-rdc each carries its own device code)
$(OBJ)/%.o: $(CSRC)/%.hip $(HEADERS) Makefile
	@mkdir -p $(@D)
	$(HIPCC) $(HIPFLAGS) -c -o $@ $<

$(OBJ)/%.o: $(CSRC)/%.cpp $(HEADERS) Makefile
	@mkdir -p $(@D)
	$(HIPCC) --offload-arch=$(ARCH) -O3 -std=c++17 -fPIC -Iinclude -I$(CSRC) -Wall -c -o $@ $<

$(LIB): $(OBJS)
	@mkdir -p $(@D)
	$(HIPCC) --offload-arch=$(ARCH) -shared -fPIC -o $@ $(OBJS) -ldl -lpthread

# the reference's command line over the library (tools/nvk_run.cpp): host-only C++ over the C ABI
CLI := nano_vllm_amd/nvk_run
cli: $(CLI)
$(CLI): tools/nvk_run.cpp include/nvk_paged_attn.h $(LIB)
	g++ -std=c++17 -O2 -Wall -Iinclude -o $@ tools/nvk_run.cpp -Lnano_vllm_amd -lnvk_paged_attn -Wl,-rpath,'$$ORIGIN'

# device assembly + register/occupancy report for the kernels as they are shipped (not needed to run)
asm: $(HIP_SRC:%=build/asm/%.o)
	cat $(HIP_SRC:%=build/asm/%.remarks) > build/resource_usage.txt

build/asm/%.o: $(CSRC)/%.hip $(HEADERS) Makefile
	@mkdir -p $(@D)
	$(HIPCC) $(HIPFLAGS) -save-temps=obj -c -Rpass-analysis=kernel-resource-usage -o $@ $< 2> build/asm/$*.remarks

# Host code under AddressSanitizer + UndefinedBehaviorSanitizer (CPU build only; the pool runs no GPU sanitizer):
# the block allocator, the tokenizer and the CPU checker behind tests/asan_driver.cpp, and the command line
# (its JSON reader and argument handling) as an instrumented executable over the normal library.
# tests/test_sanitizers.py builds and runs them on traces, random texts, and short / damaged input files.
SAN := -fsanitize=address,undefined -fno-sanitize-recover=undefined -fno-omit-frame-pointer -g -O1 -static-libasan
asan:
	mkdir -p build/asan
	gcc $(SAN) -std=c11 -c -o build/asan/nvk_oracle.o oracle/nvk_oracle.c
	g++ $(SAN) -static-libubsan -std=c++17 -Wall -Iinclude -I$(CSRC) -o build/asan/asan_driver tests/asan_driver.cpp tests/asan_stubs.cpp \
	    $(CSRC)/nvk_block_manager.cpp $(CSRC)/nvk_tokenizer.cpp build/asan/nvk_oracle.o -lpthread -lm
	g++ $(SAN) -static-libubsan -std=c++17 -Wall -Iinclude -o build/asan/nvk_run_asan tools/nvk_run.cpp -Lnano_vllm_amd -lnvk_paged_attn \
	    -Wl,-rpath,'$$ORIGIN/../../nano_vllm_amd'

oracle:
	$(MAKE) -C oracle oracle

ref:
	$(MAKE) -C oracle ref

clean:
	rm -f $(LIB) $(CLI)
	rm -rf build
	$(MAKE) -C oracle clean
