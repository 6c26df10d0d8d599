import ctypes,torch
L=ctypes.CDLL('/root/repo/_work/probe/dma/d.so'); L.go.restype=ctypes.c_float
L.go.argtypes=[ctypes.c_int,ctypes.c_void_p,ctypes.c_int,ctypes.c_int,ctypes.c_int,ctypes.c_int,ctypes.c_void_p]
B=1<<28
buf=torch.zeros(B+65536,dtype=torch.uint8,device='cuda'); out=torch.zeros(1024,dtype=torch.int32,device='cuda')
for stride in (0,4096,4224,11008):
    for region in (1<<16,1<<18,1<<20,1<<21,1<<26):
        if stride and region< (1<<20): continue
        it=400
        for g in (256,512):
            r=[]
            for kind in (0,1):
                t=L.go(kind,buf.data_ptr(),region,stride,it,g,out.data_ptr())
                r.append(g*it*64*1024/t/1e9)
            print('stride',stride,'region',region,'grid',g,'dma %.1f reg %.1f TB/s'%tuple(r),flush=True)
